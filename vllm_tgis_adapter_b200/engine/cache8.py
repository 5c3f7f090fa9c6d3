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


# (Every check is an `if` of its own: a message made for a helper's argument costs more than the launch.)
def _not_ints(x: torch.Tensor, dim: int, device: torch.device) -> bool:
    return x.dtype != torch.int32 or x.dim() != dim or x.device != device or not x.is_contiguous()


def _bad_ints(name: str, dim: int, device: torch.device) -> ValueError:
    return ValueError(f"{name}: a contiguous int32 tensor of {dim} dimension(s) on {device} is wanted")


def _pitch(name: str, x: torch.Tensor, device: torch.device) -> int:
    """Row pitch of a 2-D bf16 tensor with contiguous rows."""
    if x.dtype != torch.bfloat16 or x.dim() != 2 or x.device != device:
        raise ValueError(f"{name}: a bf16 tensor [rows, numbers] on {device} is wanted")
    rows, width = x.shape
    pitch, step = x.stride()
    if step != 1 and width > 1:
        raise ValueError(f"{name}: contiguous rows are wanted")
    return pitch if rows > 1 else width


class Cache8:
    """`pages` uint8 [n_pages, n_kv, PAGE_BYTES], zeros before the first row is written; slot = page * 32 + place."""

    def __init__(self, pages: torch.Tensor):
        if pages.dtype != torch.uint8 or pages.dim() != 3 or pages.shape[2] != PAGE_BYTES or not pages.is_cuda or not pages.is_contiguous() or pages.numel() == 0:
            raise ValueError(f"pages: a contiguous uint8 CUDA tensor [n_pages, n_kv, {PAGE_BYTES}] is wanted")
        self._lib = lib = _lib.load_library()
        self._write, self._read, self._attention, self._workspace = lib.tgis_kv8_write, lib.tgis_kv8_read, lib.tgis_kv8_attention, lib.tgis_kv8_attention_workspace
        self.pages, self.device = pages, pages.device
        self.n_pages, self.n_kv = pages.shape[0], pages.shape[1]
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)

    @classmethod
    def empty(cls, n_pages: int, n_kv: int, device: torch.device | str | None = None) -> "Cache8":
        return cls(torch.zeros(n_pages, n_kv, PAGE_BYTES, dtype=torch.uint8, device=device or "cuda"))

    def _run(self, function, *args) -> None:
        index = self.device.index
        if torch.cuda.current_device() == index:
            rc = function(self.pages.data_ptr(), self.n_pages, self.n_kv, *args, self.status.data_ptr(), torch._C._cuda_getCurrentRawStream(index))
        else:
            with torch.cuda.device(index):
                rc = function(self.pages.data_ptr(), self.n_pages, self.n_kv, *args, self.status.data_ptr(), torch._C._cuda_getCurrentRawStream(index))
        if rc != 0:
            raise ValueError(self._error())

    def _error(self) -> str:
        return (self._lib.tgis_kv8_last_error() or b"").decode(errors="replace")

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
        device = self.device
        ld = _pitch("qkv", qkv, device)
        T, width = qkv.shape
        n_q = width // HEAD_DIM - 2 * self.n_kv
        if width % HEAD_DIM != 0 or n_q < 0:
            raise ValueError(f"qkv: rows of {width} numbers are no query heads and twice {self.n_kv} heads of {HEAD_DIM}")
        if _not_ints(positions, 1, device) or positions.shape[0] != T:
            raise ValueError(f"positions: {T} contiguous int32 numbers on {device} are wanted")
        if _not_ints(slots, 1, device) or slots.shape[0] != T:
            raise ValueError(f"slots: {T} contiguous int32 numbers on {device} are wanted")
        if cos_sin.dtype != torch.bfloat16 or cos_sin.dim() != 2 or cos_sin.shape[1] != HEAD_DIM or cos_sin.device != device or not cos_sin.is_contiguous():
            raise ValueError(f"cos_sin: a contiguous bf16 tensor [positions, {HEAD_DIM}] on {device} is wanted")
        ldq = q_at = None
        if q_out is None:
            if want_q and n_q > 0:
                q_out = torch.empty((T, n_q * HEAD_DIM), dtype=torch.bfloat16, device=device)
                ldq, q_at = n_q * HEAD_DIM, q_out.data_ptr()
        else:
            ldq, q_at = _pitch("q_out", q_out, device), q_out.data_ptr()
            if q_out.shape[0] != T or q_out.shape[1] != n_q * HEAD_DIM:
                raise ValueError(f"q_out: [{T}, {n_q * HEAD_DIM}] is wanted")
        if T:
            self._run(self._write, qkv.data_ptr(), ld, T, n_q, positions.data_ptr(), slots.data_ptr(), cos_sin.data_ptr(), cos_sin.shape[0], q_at, ldq or 0)
        return q_out

    def read(self, slots: torch.Tensor, k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The rows at `slots` [T] as bf16, keys and values [T, n_kv * 128] (slots < 0: zeros)."""
        device, width = self.device, self.n_kv * HEAD_DIM
        if _not_ints(slots, 1, device):
            raise _bad_ints("slots", 1, device)
        T = slots.shape[0]
        if k_out is None:
            k_out, ldk = torch.empty((T, width), dtype=torch.bfloat16, device=device), width
        else:
            ldk = _pitch("k_out", k_out, device)
        if v_out is None:
            v_out, ldv = torch.empty((T, width), dtype=torch.bfloat16, device=device), width
        else:
            ldv = _pitch("v_out", v_out, device)
        if k_out.shape != (T, width) or v_out.shape != (T, width):
            raise ValueError(f"k_out, v_out: [{T}, {width}] are wanted")
        if T:
            self._run(self._read, slots.data_ptr(), T, k_out.data_ptr(), ldk, v_out.data_ptr(), ldv)
        return k_out, v_out

    def workspace_bytes(self, T: int, n_seqs: int, n_q: int, max_q: int, max_kv: int) -> int:
        """What `attend` needs for these bounds (no fewer for more sequences, more queries of one or longer ones; 43 MB at most)."""
        if max_q >> 31 or max_kv >> 31:   # (a longer number would be cut to 32 bits on its way)
            raise ValueError(f"max_q {max_q}, max_kv {max_kv}: numbers of 31 bits are wanted")
        n = self._workspace(T, n_seqs, n_q, self.n_kv, max_q, max_kv)
        if n < 0:
            raise ValueError(self._error())
        return n

    def attend(self, q: torch.Tensor, seqs: torch.Tensor, block_table: torch.Tensor, scale: float, max_q: int, max_kv: int, out: torch.Tensor | None = None,
               tree: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of `q` [T, n_q * 128]: `seqs` int32 [n, 4] of (first query row, queries, tokens in all, row of `block_table`), the queries
        being the last tokens of their sequence; no sequence has more than max_q queries or max_kv tokens.  A query sees what is at or
        before its place; with `tree` (int64 [T]) the queries are drafted nodes and query t sees what was there before the draft and the nodes
        whose bits are set in tree[t].  Rows that no sequence names are left as they are in `out` (undefined in a new one).
        `workspace`: a uint8 tensor of workspace_bytes(...), not shared with a call that may run at the same time; None: a new one."""
        device = self.device
        ldq = _pitch("q", q, device)
        T, width = q.shape
        if width % HEAD_DIM != 0 or width == 0:
            raise ValueError(f"q: rows of {width} numbers are no heads of {HEAD_DIM}")
        n_q = width // HEAD_DIM
        if _not_ints(seqs, 2, device) or seqs.shape[1] != 4:
            raise ValueError(f"seqs: a contiguous int32 tensor [sequences, 4] on {device} is wanted")
        if _not_ints(block_table, 2, device):
            raise _bad_ints("block_table", 2, device)
        if out is None:
            out, ldo = torch.empty((T, width), dtype=torch.bfloat16, device=device), width
        else:
            ldo = _pitch("out", out, device)
            if out.shape != q.shape:
                raise ValueError(f"out: {list(q.shape)} is wanted")
        words = None
        if tree is not None:
            if tree.dtype not in (torch.int64, torch.uint64) or tree.dim() != 1 or tree.shape[0] != T or tree.device != device or not tree.is_contiguous():
                raise ValueError(f"tree: {T} contiguous 64-bit words on {device} are wanted")
            words = tree.data_ptr()
        if max_q >> 31 or max_kv >> 31:
            raise ValueError(f"max_q {max_q}, max_kv {max_kv}: numbers of 31 bits are wanted")
        n_seqs, room, space = seqs.shape[0], 0, None
        if workspace is None:
            room = self.workspace_bytes(T, n_seqs, n_q, max_q, max_kv)
            if room:
                workspace = torch.empty(room, dtype=torch.uint8, device=device)   # (the stream's: the next call's may be the same memory)
                space = workspace.data_ptr()
        else:
            if workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.device != device:
                raise ValueError(f"workspace: a contiguous uint8 tensor on {device} is wanted")
            room, space = workspace.numel(), workspace.data_ptr()
        if T and n_seqs:
            self._run(self._attention, q.data_ptr(), ldq, T, n_q, seqs.data_ptr(), n_seqs, block_table.data_ptr(), block_table.shape[0], block_table.shape[1], words,
                      scale, max_q, max_kv, out.data_ptr(), ldo, space, room)
        return out
