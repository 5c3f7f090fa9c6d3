"""Products with 8-bit weights (csrc/rows8.cu, csrc/gemm8.cu; C ABI: include/tgis_w8.h).

    layer = Linear8.from_weight(w)                    # w [n, k]: every block of 128 x 128 as e4m3 codes with one fp32 scale
    rows = quantise(x)                                # x [T, k]: every 128 neighbours of a row as e4m3 codes with one fp32 scale
    rows = quantise(x, norm=w_norm, residual=res)     # ... of the RMS norm of x + residual, which is updated
    y = layer(rows)                                   # [T, n]
    y = FeedForward8(gate, up, down)(rows)            # silu(gate x) * (up x) in 8-bit rows, then the down projection

`Linear8(codes, scales)` takes a checkpoint's block-scaled matrix as it is.  Calls go to the current stream of their tensors' device and return
after the launch; they may be captured into CUDA graphs and, having no workspace, run at the same time.  Results do not take the place of what they are
made of, the residual's sum excepted.  Arguments that the host can check raise ValueError.
"""
from __future__ import annotations

import ctypes as C
import threading

import torch

from . import _lib
from ._lib import TgisW8Matrix, TgisW8Rows

GROUP, MAX_K, MAX_ROWS = 128, 131072, 1 << 22
TYPES = {torch.bfloat16: 0, torch.float32: 1}
NOT_ROWS = "x: rows in 8 bits are wanted (Rows8, of quantise)"
_functions = None
_lock = threading.Lock()   # of what is made once a device, and of the status words' counts
_current_device, _stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


class _Functions:
    def __init__(self):
        lib = _lib.load_library()
        self.rows, self.weight, self.product, self.gated, self.feed_forward = (
            lib.tgis_w8_quantise_rows, lib.tgis_w8_quantise_weight, lib.tgis_w8_product, lib.tgis_w8_gated, lib.tgis_w8_feed_forward)
        self.error = lib.tgis_w8_last_error


def _load() -> _Functions:
    global _functions
    if _functions is None:
        _functions = _Functions()
    return _functions


def _run(function, device: torch.device, *args) -> None:
    index = device.index
    if _current_device() == index:
        rc = function(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = function(*args, _stream(index))
    if rc != 0:
        raise ValueError((_load().error() or b"").decode(errors="replace"))


def _pitch(name: str, x: torch.Tensor, device: torch.device | None = None) -> int:
    """Row pitch of a 2-D bf16 or fp32 CUDA tensor with contiguous rows."""
    shape = x.shape
    if x.dtype not in TYPES or len(shape) != 2 or not x.is_cuda or (device is not None and x.device != device):
        raise ValueError(f"{name}: a bf16 or fp32 tensor [rows, numbers] on {device or 'a CUDA device'} is wanted")
    rows, width = shape
    pitch, step = x.stride()
    if step != 1 and width > 1:
        raise ValueError(f"{name}: contiguous rows are wanted")
    return pitch if rows > 1 else width


class _Device:
    """What calls on a device share: empty tensors, whose new_empty costs half of torch.empty's time, and the status word."""

    def __init__(self, device: torch.device):
        self.device, self.status, self.status_at, self.stalls = device, None, None, 0
        self.fp32, self.bf16, self.codes, self.bytes = (torch.empty(0, dtype=t, device=device) for t in (torch.float32, torch.bfloat16, torch.float8_e4m3fn, torch.uint8))

    def with_status(self) -> "_Device":
        if self.status_at is None:
            with _lock:
                if self.status_at is None:
                    if torch.cuda.is_current_stream_capturing():   # (the word would be a graph's, and zeroed by its replays)
                        raise ValueError("the first layer on a device is made before a capture begins")
                    with torch.cuda.device(self.device):
                        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
                        torch.cuda.current_stream().synchronize()
                    self.status_at = self.status.data_ptr()
        return self

    def stalls_so_far(self) -> int:
        """How often a check has found the word raised, with this one, which waits for the device.  The word is taken back here and the count is what a layer
        compares with what it saw last, so that no check takes another layer's report."""
        with torch.cuda.device(self.device):
            torch.cuda.synchronize()
            with _lock:
                if int(self.status.item()):
                    self.status.zero_()
                    torch.cuda.current_stream().synchronize()
                    self.stalls += 1
                return self.stalls


_devices: dict[int, _Device] = {}


def _of(device: torch.device) -> _Device:
    got = _devices.get(device.index)
    if got is None:
        made = _Device(device)
        with _lock:
            got = _devices.setdefault(device.index, made)
    return got


class _Checked:
    """A layer's check; `_watch` when it is made."""

    def _watch(self, on: _Device) -> None:
        self._on, self._seen = on, on.stalls

    def check(self) -> None:
        """Waits for the device and raises if a call on it, whichever layer's, has given up since this layer's last check."""
        stalls = self._on.stalls_so_far()
        seen, self._seen = self._seen, stalls
        if stalls != seen:
            raise RuntimeError("a wait inside a kernel ran out")


class Rows8:
    """T rows of k numbers in 8 bits: `codes` e4m3 [T, k], `scales` fp32 [groups, T]; views of tensors whose rows are as long as whole groups are."""

    __slots__ = ("codes", "scales", "device", "record", "at")

    def __init__(self, T: int, k: int, device: torch.device):
        if device.index is None:
            device = torch.device(device.type, torch.cuda.current_device())
        groups, on = -(-k // GROUP), _of(device)
        codes, scales = on.codes.new_empty((T, groups * GROUP)), on.fp32.new_empty((groups, T))
        self.device = device
        self.record = TgisW8Rows(codes.data_ptr(), scales.data_ptr(), groups * GROUP, T, T, k)
        self.at = C.addressof(self.record)
        self.codes, self.scales = codes if k == groups * GROUP else codes[:, :k], scales

    @property
    def shape(self) -> tuple[int, int]:
        return self.record.t, self.record.k

    def values(self) -> torch.Tensor:
        """What the rows stand for, fp32 [T, k]."""
        return self.codes.float() * self.scales.t().repeat_interleave(GROUP, dim=1)[:, : self.codes.shape[1]]


def quantise(x: torch.Tensor, norm: torch.Tensor | None = None, eps: float = 1e-5, residual: torch.Tensor | None = None,
             residual_out: torch.Tensor | None = None, out: Rows8 | None = None) -> Rows8:
    """Rows of x [T, k] (bf16 or fp32) in 8 bits.  `residual` (like x): x + residual, rounded to their type, takes the place of x and is stored in
    `residual_out` (None: residual itself; x will do).  `norm` (bf16 [k]): the RMS norm's weight, v = r * norm / sqrt(mean r^2 + eps)."""
    ld = _pitch("x", x)
    device, dtype, shape = x.device, x.dtype, x.shape
    T, k = shape
    if k < 1 or k > MAX_K or T > MAX_ROWS:
        raise ValueError(f"x: at most {MAX_ROWS} rows of 1 to {MAX_K} numbers are wanted, not {T} of {k}")
    norm_at = res_at = to_at = None
    ldr = ldt = 0
    if norm is not None:
        if norm.dtype != torch.bfloat16 or norm.shape != (k,) or norm.device != device or not norm.is_contiguous():
            raise ValueError(f"norm: {k} contiguous bf16 numbers on {device} are wanted")
        norm_at = norm.data_ptr()
    if residual is not None:
        ldr = _pitch("residual", residual, device)
        if residual_out is None:
            residual_out, ldt = residual, ldr
        else:
            ldt = _pitch("residual_out", residual_out, device)
        if residual.shape != shape or residual.dtype != dtype or residual_out.shape != shape or residual_out.dtype != dtype:
            raise ValueError(f"residual, residual_out: {dtype} tensors [{T}, {k}] are wanted")
        res_at, to_at = residual.data_ptr(), residual_out.data_ptr()
    elif residual_out is not None:
        raise ValueError("residual_out: there is no residual")
    if out is None:
        out = Rows8(T, k, device)
    elif not isinstance(out, Rows8) or out.shape != (T, k) or out.device != device:
        raise ValueError(f"out: {T} rows of {k} numbers on {device} are wanted")
    if T or norm is not None:
        _run(_load().rows, device, x.data_ptr(), TYPES[dtype], ld, norm_at, eps, res_at, ldr, to_at, ldt, out.at)
    return out


class Linear8(_Checked):
    """A weight matrix in 8 bits: `codes` e4m3 [n, k], `scales` fp32 [blocks of 128 rows, groups of 128].  Codes whose rows do not start on
    16 bytes are copied once."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype != torch.float8_e4m3fn or codes.dim() != 2 or not codes.is_cuda or codes.numel() == 0:
            raise ValueError("codes: a torch.float8_e4m3fn CUDA tensor [n, k] is wanted")
        n, k = codes.shape
        blocks = (-(-n // GROUP), -(-k // GROUP))
        if k > MAX_K or n > MAX_ROWS:
            raise ValueError(f"codes: at most {MAX_ROWS} rows of {MAX_K} numbers are wanted, not {n} of {k}")
        if scales.dtype != torch.float32 or tuple(scales.shape) != blocks or scales.device != codes.device or not scales.is_contiguous():
            raise ValueError(f"scales: a contiguous fp32 tensor {list(blocks)} on {codes.device} is wanted")
        pitch, step = codes.stride()
        if n == 1:
            pitch = -(-k // 16) * 16
        if (step != 1 and k > 1) or pitch < k or pitch % 16 or codes.data_ptr() % 16:
            rows = torch.zeros((n, blocks[1] * GROUP), dtype=torch.uint8, device=codes.device)
            rows[:, :k] = codes.view(torch.uint8)
            codes, pitch = rows.view(torch.float8_e4m3fn)[:, :k], blocks[1] * GROUP
        self._keep(codes, scales, codes.device, TgisW8Matrix(codes.data_ptr(), scales.data_ptr(), pitch, n, k))

    def _keep(self, codes: torch.Tensor, scales: torch.Tensor, device: torch.device, record: TgisW8Matrix) -> None:
        self.codes, self.scales, self.device, self.n, self.k = codes, scales, device, record.n, record.k
        self.record, self.at = record, C.addressof(record)
        self._watch(_of(device).with_status())
        self._product = _load().product

    @classmethod
    def from_weight(cls, w: torch.Tensor) -> "Linear8":
        """w [n, k] (bf16 or fp32) in 8 bits."""
        ld = _pitch("w", w)
        n, k = w.shape
        if w.numel() == 0 or k > MAX_K or n > MAX_ROWS:
            raise ValueError(f"w: 1 to {MAX_ROWS} rows of 1 to {MAX_K} numbers are wanted, not {n} of {k}")
        groups = -(-k // GROUP)
        on = _of(w.device)
        codes, scales = on.codes.new_empty((n, groups * GROUP)), on.fp32.new_empty((-(-n // GROUP), groups))
        made = cls.__new__(cls)
        made._keep(codes if k == groups * GROUP else codes[:, :k], scales, w.device, TgisW8Matrix(codes.data_ptr(), scales.data_ptr(), groups * GROUP, n, k))
        _run(_load().weight, made.device, w.data_ptr(), TYPES[w.dtype], ld, made.at)
        return made

    def values(self) -> torch.Tensor:
        """What the matrix stands for, fp32 [n, k]."""
        s = self.scales.repeat_interleave(GROUP, dim=0)[: self.n].repeat_interleave(GROUP, dim=1)[:, : self.k]
        return self.codes.float() * s

    def __call__(self, x: Rows8, out: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """x w^T [T, n], in `dtype` (bf16 or fp32) or into `out`."""
        if not isinstance(x, Rows8):
            raise ValueError(NOT_ROWS)
        T, k = x.record.t, x.record.k
        if k != self.k or x.device != self.device:
            raise ValueError(f"x: rows of {self.k} numbers on {self.device} are wanted, not of {k} on {x.device}")
        out, ld = _result(out, dtype, T, self.n, self._on, self.device)
        if T:
            _run(self._product, self.device, x.at, self.at, out.data_ptr(), TYPES[out.dtype], ld, self._on.status_at)
        return out


def _result(out: torch.Tensor | None, dtype: torch.dtype, T: int, n: int, on: _Device, device: torch.device) -> tuple[torch.Tensor, int]:
    if out is None:
        if dtype not in TYPES:
            raise ValueError("dtype: torch.bfloat16 or torch.float32 is wanted")
        return (on.bf16 if dtype == torch.bfloat16 else on.fp32).new_empty((T, n)), n
    ld = _pitch("out", out, device)
    if out.shape[0] != T or out.shape[1] != n:
        raise ValueError(f"out: [{T}, {n}] is wanted")
    return out, ld


class FeedForward8(_Checked):
    """y = down h, h = silu(gate x) * (up x) held in 8-bit rows between the two launches."""

    def __init__(self, gate: Linear8, up: Linear8, down: Linear8):
        if not all(isinstance(m, Linear8) for m in (gate, up, down)):
            raise ValueError("gate, up, down: 8-bit matrices are wanted (Linear8)")
        if up.n != gate.n or up.k != gate.k or down.k != gate.n or up.device != gate.device or down.device != gate.device:
            raise ValueError(f"gate [{gate.n}, {gate.k}], up [{up.n}, {up.k}], down [{down.n}, {down.k}] on one device do not make a feed-forward block")
        if gate.n > MAX_K:
            raise ValueError(f"gate: at most {MAX_K} rows are wanted")
        self.gate, self.up, self.down, self.device = gate, up, down, gate.device
        self._watch(gate._on)
        self._call = _load().feed_forward
        self._groups = -(-gate.n // GROUP)

    def hidden(self, x: Rows8, out: Rows8 | None = None) -> Rows8:
        """h alone."""
        self._fits(x)
        T = x.record.t
        if out is None:
            out = Rows8(T, self.gate.n, self.device)
        elif not isinstance(out, Rows8) or out.shape != (T, self.gate.n) or out.device != self.device:
            raise ValueError(f"out: {T} rows of {self.gate.n} numbers on {self.device} are wanted")
        if T:
            _run(_load().gated, self.device, x.at, self.gate.at, self.up.at, out.at, self._on.status_at)
        return out

    def _fits(self, x: Rows8) -> None:
        if not isinstance(x, Rows8):
            raise ValueError(NOT_ROWS)
        if x.record.k != self.gate.k or x.device != self.device:
            raise ValueError(f"x: rows of {self.gate.k} numbers on {self.device} are wanted, not of {x.record.k} on {x.device}")

    def __call__(self, x: Rows8, out: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """[T, down's n], in `dtype` (bf16 or fp32) or into `out`."""
        self._fits(x)
        T = x.record.t
        out, ld = _result(out, dtype, T, self.down.n, self._on, self.device)
        if T:
            width = self._groups * GROUP
            room = self._on.bytes.new_empty(T * (width + self._groups * 4))   # (the stream's: the next call's may be the same memory)
            at = room.data_ptr()
            h = TgisW8Rows(at, at + T * width, width, T, T, self.gate.n)
            _run(self._call, self.device, x.at, self.gate.at, self.up.at, self.down.at, C.addressof(h), out.data_ptr(), TYPES[out.dtype], ld, self._on.status_at)
        return out
