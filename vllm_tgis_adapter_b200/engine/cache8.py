"""The 8-bit paged cache of one layer and the attention that reads it (csrc/cache8.cu, csrc/attention8.cu; C ABI: include/tgis_kv8.h).

    cache = Cache8.empty(n_pages, n_kv)
    q = cache.write(qkv, positions, slots, cos_sin)                  # rotate, quantise, scatter
    out = cache.attend(q, seqs, block_table, scale, max_q, max_kv)   # single tokens, prompts' portions; tree=words: drafted trees
    k, v = cache.read(slots)                                         # rows as bf16

The engine stores its cache like this under `kv_cache_dtype="fp8"`.  Calls go to the current stream of the cache's device and return
after the launch; they may be captured into CUDA graphs.  Arguments that the host can check raise ValueError; what only the device
sees (slots, pages, records) is left out there and reported by `check()`.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

PAGE_TOKENS, HEAD_DIM, PAGE_BYTES, MAX_TREE, MAX_SEQS = 32, 128, 8448, 64, 4096
BAD = {1: "a slot behind the last page", 2: "a position outside the rotation table", 4: "a sequence record that contradicts the call",
       8: "a page number outside the cache", 16: "a wait inside a kernel ran out"}


def _want(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _ints(name: str, x: torch.Tensor, dim: int, device: torch.device) -> None:
    _want(x.dtype == torch.int32 and x.dim() == dim and x.device == device and x.is_contiguous(),
          f"{name}: a contiguous int32 tensor of {dim} dimension(s) on {device} is wanted")


def _rows(name: str, x: torch.Tensor, device: torch.device) -> int:
    """Row pitch of a 2-D bf16 tensor with contiguous rows."""
    _want(x.dtype == torch.bfloat16 and x.dim() == 2 and x.device == device and (x.shape[1] == 1 or x.stride(1) == 1),
          f"{name}: a bf16 tensor [rows, numbers] with contiguous rows on {device} is wanted")
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


class Cache8:
    """`pages` uint8 [n_pages, n_kv, PAGE_BYTES], zeros before the first row is written; slot = page * 32 + place."""

    def __init__(self, pages: torch.Tensor):
        _want(pages.dtype == torch.uint8 and pages.dim() == 3 and pages.shape[2] == PAGE_BYTES and pages.is_cuda and pages.is_contiguous() and pages.numel() > 0,
              f"pages: a contiguous uint8 CUDA tensor [n_pages, n_kv, {PAGE_BYTES}] is wanted")
        self._call = _lib.load_library()
        self.pages, self.device = pages, pages.device
        self.n_pages, self.n_kv = pages.shape[0], pages.shape[1]
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)

    @classmethod
    def empty(cls, n_pages: int, n_kv: int, device: torch.device | str | None = None) -> "Cache8":
        return cls(torch.zeros(n_pages, n_kv, PAGE_BYTES, dtype=torch.uint8, device=device or "cuda"))

    def _run(self, function, *args) -> None:
        index = self.device.index
        if torch.cuda.current_device() == index:
            rc = function(*args, self.status.data_ptr(), torch._C._cuda_getCurrentRawStream(index))
        else:
            with torch.cuda.device(index):
                rc = function(*args, self.status.data_ptr(), torch._C._cuda_getCurrentRawStream(index))
        if rc != 0:
            raise ValueError((self._call.tgis_kv8_last_error() or b"").decode(errors="replace"))

    def check(self) -> None:
        """Waits for the device and raises if a call since the last check met something that it left out."""
        with torch.cuda.device(self.device):
            torch.cuda.synchronize()
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise RuntimeError("; ".join(text for bit, text in BAD.items() if bits & bit))

    def write(self, qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, cos_sin: torch.Tensor,
              q_out: torch.Tensor | None = None, want_q: bool = True) -> torch.Tensor | None:
        """Queries and keys of `qkv` [T, (n_q + 2 n_kv) * 128] rotated at `positions`, keys and values stored at `slots` (< 0: not
        stored; the others differ).  Returns the rotated queries [T, n_q * 128] (None where not wanted, or n_q == 0)."""
        ld = _rows("qkv", qkv, self.device)
        T, width = qkv.shape
        n_q = width // HEAD_DIM - 2 * self.n_kv
        _want(width % HEAD_DIM == 0 and n_q >= 0, f"qkv: rows of {width} numbers are no query heads and twice {self.n_kv} heads of {HEAD_DIM}")
        _ints("positions", positions, 1, self.device)
        _ints("slots", slots, 1, self.device)
        _want(positions.shape[0] == T and slots.shape[0] == T, f"positions, slots: {T} are wanted")
        _want(cos_sin.dtype == torch.bfloat16 and cos_sin.dim() == 2 and cos_sin.shape[1] == HEAD_DIM and cos_sin.device == self.device and cos_sin.is_contiguous(),
              f"cos_sin: a contiguous bf16 tensor [positions, {HEAD_DIM}] on {self.device} is wanted")
        if q_out is None and want_q and n_q > 0:
            q_out = torch.empty(T, n_q * HEAD_DIM, dtype=torch.bfloat16, device=self.device)
        ldq = 0
        if q_out is not None:
            ldq = _rows("q_out", q_out, self.device)
            _want(q_out.shape[0] == T and q_out.shape[1] == n_q * HEAD_DIM, f"q_out: [{T}, {n_q * HEAD_DIM}] is wanted")
        if T:
            self._run(self._call.tgis_kv8_write, self.pages.data_ptr(), self.n_pages, self.n_kv, qkv.data_ptr(), ld, T, n_q, positions.data_ptr(),
                      slots.data_ptr(), cos_sin.data_ptr(), cos_sin.shape[0], q_out.data_ptr() if q_out is not None else None, ldq)
        return q_out

    def read(self, slots: torch.Tensor, k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The rows at `slots` [T] as bf16, keys and values [T, n_kv * 128] (slots < 0: zeros)."""
        _ints("slots", slots, 1, self.device)
        T, width = slots.shape[0], self.n_kv * HEAD_DIM
        k_out = torch.empty(T, width, dtype=torch.bfloat16, device=self.device) if k_out is None else k_out
        v_out = torch.empty(T, width, dtype=torch.bfloat16, device=self.device) if v_out is None else v_out
        ldk, ldv = _rows("k_out", k_out, self.device), _rows("v_out", v_out, self.device)
        _want(k_out.shape == (T, width) and v_out.shape == (T, width), f"k_out, v_out: [{T}, {width}] are wanted")
        if T:
            self._run(self._call.tgis_kv8_read, self.pages.data_ptr(), self.n_pages, self.n_kv, slots.data_ptr(), T, k_out.data_ptr(), ldk, v_out.data_ptr(), ldv)
        return k_out, v_out

    def workspace_bytes(self, T: int, n_seqs: int, n_q: int, max_q: int, max_kv: int) -> int:
        """What `attend` needs for these bounds (no fewer for larger ones of the same kind of call)."""
        n = self._call.tgis_kv8_attention_workspace(T, n_seqs, n_q, self.n_kv, max_q, max_kv)
        if n < 0:
            raise ValueError((self._call.tgis_kv8_last_error() or b"").decode(errors="replace"))
        return n

    def attend(self, q: torch.Tensor, seqs: torch.Tensor, block_table: torch.Tensor, scale: float, max_q: int, max_kv: int, out: torch.Tensor | None = None,
               tree: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of `q` [T, n_q * 128]: `seqs` int32 [n, 4] of (first query row, queries, tokens in all, row of `block_table`), the queries
        being the last tokens of their sequence; no sequence has more than max_q queries or max_kv tokens.  A query sees what is at or
        before its place; with `tree` (int64 [T]) the queries are drafted nodes and query t sees what was there before the draft and the nodes
        whose bits are set in tree[t].  Rows that no sequence names are left as they are in `out` (undefined in a new one).
        `workspace`: a uint8 tensor of workspace_bytes(...), not shared with a call that may run at the same time; None: a new one."""
        ldq = _rows("q", q, self.device)
        T, width = q.shape
        _want(width % HEAD_DIM == 0 and width > 0, f"q: rows of {width} numbers are no heads of {HEAD_DIM}")
        n_q = width // HEAD_DIM
        _ints("seqs", seqs, 2, self.device)
        _ints("block_table", block_table, 2, self.device)
        _want(seqs.shape[1] == 4, "seqs: four numbers a sequence are wanted")
        if out is None:
            out = torch.empty(T, width, dtype=torch.bfloat16, device=self.device)
        ldo = _rows("out", out, self.device)
        _want(out.shape == q.shape, f"out: {list(q.shape)} is wanted")
        if tree is not None:
            _want(tree.dtype in (torch.int64, torch.uint64) and tree.dim() == 1 and tree.shape[0] == T and tree.device == self.device and tree.is_contiguous(),
                  f"tree: {T} contiguous 64-bit words on {self.device} are wanted")
        need = self.workspace_bytes(T, seqs.shape[0], n_q, max_q, max_kv)
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        else:
            _want(workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.device == self.device, f"workspace: a contiguous uint8 tensor on {self.device} is wanted")
        if T and seqs.shape[0]:
            self._run(self._call.tgis_kv8_attention, self.pages.data_ptr(), self.n_pages, self.n_kv, q.data_ptr(), ldq, T, n_q, seqs.data_ptr(), seqs.shape[0],
                      block_table.data_ptr(), block_table.shape[0], block_table.shape[1], tree.data_ptr() if tree is not None else None, scale, max_q, max_kv,
                      out.data_ptr(), ldo, workspace.data_ptr() if workspace is not None else None, workspace.numel() if workspace is not None else 0)
        return out
