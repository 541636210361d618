"""Functional API over libfrag.so for torch CUDA tensors.

Every op validates dtypes/shapes on the host, allocates its outputs (and any
workspace) with torch on the input's device, and launches the CUDA kernels
through the C ABI on the current stream.  Nothing here computes on the CPU:
if the library is missing the call raises.

Embedding ids are range-checked on the device.  A bad id writes a zero row and
sets a flag in a per-device status word; ``check_status()`` synchronises and
raises ``IndexError`` if any flag is set.  Set ``FRAG_SYNC_CHECK=1`` to check
after every embedding call (what torch's device-side assert would catch).
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import operator
import os
import warnings
from array import array

import torch

from . import _lib
from ._lib import FragError

__all__ = [
    "FragError",
    "rmsnorm_fwd",
    "add_rmsnorm_fwd",
    "rmsnorm_bwd",
    "rmsnorm_fwd_bwd",
    "rmsnorm_bwd_workspace_bytes",
    "rmsnorm_bwd_num_blocks",
    "dw_reduce",
    "embedding_fwd",
    "embedding_rmsnorm_fwd",
    "embedding_bwd",
    "rmsnorm_embedding_bwd",
    "copy_rows",
    "copy_rows_grouped",
    "convert",
    "rope",
    "rope_complex",
    "RopeFrequencies",
    "rope_scaled",
    "rmsnorm_quant_fwd",
    "rmsnorm_quant_bwd",
    "orthogonalize",
    "muon_update",
    "orthogonalize_workspace_bytes",
    "layernorm_fwd",
    "layernorm_bwd",
    "grad_norm",
    "AdamWStates",
    "adamw_update",
    "check_status",
    "reset_status",
]

_SYNC_CHECK = os.environ.get("FRAG_SYNC_CHECK", "0") not in ("", "0")
_status_words: dict[int, torch.Tensor] = {}


# These helpers run in every call, and a small call's time is the host's: a raw
# stream handle takes 0.1 us where a Stream object takes 2.5, a plain class
# 0.5 us where a generator context takes 1.3.

def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _stream(dev: torch.device):
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if dev.index is None else dev.index)


def _new(like: torch.Tensor, shape, dtype: torch.dtype) -> torch.Tensor:
    """A new tensor on like's device (one integer size: 1.6 us, a tuple: 2.5)."""
    return like.new_empty(shape[0] if len(shape) == 1 else shape, dtype=dtype)


class _on_device:
    """Makes `dev` the current CUDA device for a with block."""

    __slots__ = ("idx", "prev")

    def __init__(self, dev: torch.device):
        if dev.type != "cuda":
            raise ValueError(f"kernelproblems_b200 ops need CUDA tensors, got device {dev}")
        self.idx = dev.index

    def __enter__(self):
        cur = torch.cuda.current_device()
        self.prev = None
        if self.idx is not None and self.idx != cur:
            self.prev = cur
            torch.cuda.set_device(self.idx)

    def __exit__(self, *exc):
        if self.prev is not None:
            torch.cuda.set_device(self.prev)


def _need(t: torch.Tensor, name: str, dtype: torch.dtype, dev: torch.device | None = None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if dev is not None and t.device != dev:
        raise ValueError(f"{name} is on {t.device}, expected {dev}")


def _check_out(t: torch.Tensor, name: str, dtype: torch.dtype, dev: torch.device, *,
               shape: tuple | None = None, numel: int | None = None) -> torch.Tensor:
    """A caller-supplied output buffer is written by the kernel as one dense
    block of `shape` (or `numel` elements), so it must be exactly that: the
    right shape or element count, dtype and device, and contiguous.  Anything
    else would let the kernel write past the buffer."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: shape {tuple(t.shape)} != {tuple(shape)}")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name}: {t.numel()} elements, the kernel writes {numel}")
    if t.dtype != dtype:
        raise ValueError(f"{name}: dtype {t.dtype} != {dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, expected {dev}")
    return t


def _status_word(dev: torch.device) -> torch.Tensor:
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    w = _status_words.get(idx)
    if w is None:
        w = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", idx))
        _status_words[idx] = w
    return w


def check_status(device: torch.device | int | None = None) -> None:
    """Synchronise and raise IndexError if a kernel flagged an out-of-range id
    (embedding ids, RoPE table positions),
    RuntimeError if a kernel gave up waiting for its own copies (a bounded
    wait expired: its outputs are not valid)."""
    lib = _lib.load()
    cur = torch.cuda.current_device()
    dev_idx = cur if device is None else (device if isinstance(device, int) else device.index)
    with torch.cuda.device(dev_idx if dev_idx is not None else cur):
        flags = lib.frag_device_errors(1)
    if flags < 0:
        raise FragError("frag_device_errors", -flags)
    if flags & _lib.FRAG_DEVFLAG_WAIT_TIMEOUT:
        raise RuntimeError("a libfrag kernel's bounded wait expired; its outputs are invalid")
    if flags & _lib.FRAG_DEVFLAG_INDEX_OOB:
        raise IndexError("rope: a position was outside the freqs table")
    if device is None:
        devs = list(_status_words)
    elif isinstance(device, int):
        devs = [device]
    else:  # torch.device("cuda") without an index means the current device
        devs = [device.index if device.index is not None else cur]
    for idx in devs:
        w = _status_words.get(idx)
        if w is None:
            continue
        v = int(w.item())
        if v & _lib.FRAG_DEVFLAG_INDEX_OOB:
            w.zero_()
            raise IndexError("embedding: an index was outside [0, num_embeddings)")


def reset_status() -> None:
    for w in _status_words.values():
        w.zero_()


# ---------------------------------------------------------------- RMSNorm

def _rows(x: torch.Tensor, N: int, name: str) -> int:
    if x.shape[-1] != N:
        raise ValueError(f"{name}: last dim {x.shape[-1]} != normalized size {N}")
    if not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return x.numel() // N if N else 0


def rmsnorm_fwd(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *,
                out: torch.Tensor | None = None, rstd: torch.Tensor | None = None,
                save_rstd: bool = True):
    """y = bf16((x * rstd) * w), rstd = 1/sqrt(mean(x^2)+eps) per row (fp32).

    Returns (y, rstd) with y shaped like x and rstd shaped x.shape[:-1]
    (None when save_rstd is False)."""
    _need(x, "x", torch.bfloat16)
    _need(weight, "weight", torch.bfloat16, x.device)
    N = weight.numel()
    M = _rows(x, N, "x")
    y = (torch.empty_like(x) if out is None
         else _check_out(out, "out", torch.bfloat16, x.device, shape=x.shape))
    if save_rstd and rstd is None:
        rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    elif save_rstd:
        _check_out(rstd, "rstd", torch.float32, x.device, numel=M)
    wc = weight.contiguous()
    with _on_device(x.device):
        _lib.call("frag_rmsnorm_fwd", _ptr(x), _ptr(wc), _ptr(y),
                  _ptr(rstd if save_rstd else None), M, N, float(eps), _stream(x.device))
    return y, (rstd if save_rstd else None)


def add_rmsnorm_fwd(residual: torch.Tensor, x: torch.Tensor, weight: torch.Tensor,
                    eps: float = 1e-5, *, write_h: bool = True, save_rstd: bool = True,
                    h_out: torch.Tensor | None = None, y_out: torch.Tensor | None = None):
    """h = bf16(residual + x); y = rmsnorm(h) * w.  Returns (h, y, rstd)."""
    _need(residual, "residual", torch.bfloat16)
    _need(x, "x", torch.bfloat16, residual.device)
    _need(weight, "weight", torch.bfloat16, residual.device)
    if residual.shape != x.shape:
        raise ValueError(f"residual {tuple(residual.shape)} and x {tuple(x.shape)} differ")
    N = weight.numel()
    M = _rows(x, N, "x")
    _rows(residual, N, "residual")
    h = None
    if write_h:
        h = (torch.empty_like(x) if h_out is None
             else _check_out(h_out, "h_out", torch.bfloat16, x.device, shape=x.shape))
    y = (torch.empty_like(x) if y_out is None
         else _check_out(y_out, "y_out", torch.bfloat16, x.device, shape=x.shape))
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) if save_rstd else None
    wc = weight.contiguous()
    with _on_device(x.device):
        _lib.call("frag_add_rmsnorm_fwd", _ptr(residual), _ptr(x), _ptr(wc),
                  _ptr(h), _ptr(y), _ptr(rstd), M, N, float(eps), _stream(x.device))
    return h, y, rstd


def rmsnorm_fwd_bwd(x: torch.Tensor, weight: torch.Tensor, dy: torch.Tensor, *,
                    x2: torch.Tensor | None = None, x3: torch.Tensor | None = None,
                    dy2: torch.Tensor | None = None, dy3: torch.Tensor | None = None,
                    dres: torch.Tensor | None = None, eps: float = 1e-5,
                    write_y: bool = True, save_rstd: bool = False,
                    dw_dtype: torch.dtype | None = torch.float32,
                    workspace: torch.Tensor | None = None):
    """RMSNorm forward recomputed inside its backward, one pass
    (frag_rmsnorm_fwd_bwd).  Returns (y, rstd, dx, dw):

    h     bf16(bf16(x + x2) + x3) (x2, x3 optional), never written
    y     bf16((h * rstd) * w) like x, or None (write_y=False)
    rstd  fp32 [rows], or None (save_rstd=False)
    dx    bf16(dres + bf16(RMSNorm backward of bf16(bf16(dy + dy2) + dy3)))
    dw    fp32, bf16 or None, summed in a fixed order
    """
    _need(x, "x", torch.bfloat16)
    dev = x.device
    _need(weight, "weight", torch.bfloat16, dev)
    N = weight.numel()
    M = _rows(x, N, "x")
    if x3 is not None and x2 is None:
        raise ValueError("x3 needs x2 (the inputs are summed in order)")
    if dy3 is not None and dy2 is None:
        raise ValueError("dy3 needs dy2 (the gradients are summed in order)")
    for name, t in (("dy", dy), ("x2", x2), ("x3", x3), ("dy2", dy2), ("dy3", dy3), ("dres", dres)):
        if t is not None:
            _need(t, name, torch.bfloat16, dev)
            if t.shape != x.shape:
                raise ValueError(f"{name} {tuple(t.shape)} and x {tuple(x.shape)} differ")
            _rows(t, N, name)
    if dw_dtype not in (None, torch.float32, torch.bfloat16):
        raise TypeError("dw_dtype must be float32, bfloat16 or None")
    y = torch.empty_like(x) if write_y else None
    rstd = torch.empty(M, dtype=torch.float32, device=dev) if save_rstd else None
    dx = torch.empty_like(x)
    dw = None if dw_dtype is None else torch.empty(N, dtype=dw_dtype, device=dev)
    with _on_device(dev):
        lib = _lib.load()
        need = int(lib.frag_rmsnorm_bwd_workspace_bytes(M, N))
        if workspace is None or workspace.numel() < need:
            workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
        _lib.call("frag_rmsnorm_fwd_bwd", _ptr(x), _ptr(x2), _ptr(x3), _ptr(weight.contiguous()),
                  _ptr(dy), _ptr(dy2), _ptr(dy3), _ptr(dres), _ptr(y), _ptr(rstd), _ptr(dx),
                  _ptr(dw) if dw_dtype == torch.float32 else None,
                  _ptr(dw) if dw_dtype == torch.bfloat16 else None,
                  M, N, float(eps), _ptr(workspace), workspace.numel(), _stream(dev))
    return y, rstd, dx, dw


def rmsnorm_bwd_workspace_bytes(M: int, N: int, device=None) -> int:
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with _on_device(dev):
        return int(_lib.load().frag_rmsnorm_bwd_workspace_bytes(M, N))


def rmsnorm_bwd_num_blocks(M: int, N: int, device=None) -> int:
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with _on_device(dev):
        return int(_lib.load().frag_rmsnorm_bwd_num_blocks(M, N))


def rmsnorm_bwd(dy: torch.Tensor, x: torch.Tensor, rstd: torch.Tensor | None,
                weight: torch.Tensor, *, dy2: torch.Tensor | None = None,
                dy3: torch.Tensor | None = None,
                dres: torch.Tensor | None = None, eps: float = 1e-6,
                dw_dtype: torch.dtype | None = torch.float32,
                workspace: torch.Tensor | None = None, return_partials: bool = False,
                dx_out: torch.Tensor | None = None, dw_out: torch.Tensor | None = None):
    """RMSNorm backward.  Returns (dx, dw[, partials]).

    dy2   optional second gradient summed (in bf16) into dy first
    dy3   optional third gradient (needs dy2): dy = bf16(bf16(dy + dy2) + dy3)
    rstd  saved rstd (fp32, one per row) or None to recompute it with eps
    dres  optional residual gradient added (in bf16) to dx
    dw    fp32 (dw_dtype=torch.float32), bf16, or None (not reduced)
    dx_out, dw_out  optional preallocated outputs (x-shaped bf16, N elements
          of dw_dtype), written in place and returned
    partials  the [G, N] fp32 per-row-block sums, for cross-rank reductions
    """
    _need(dy, "dy", torch.bfloat16)
    dev = dy.device
    _need(x, "x", torch.bfloat16, dev)
    _need(weight, "weight", torch.bfloat16, dev)
    N = weight.numel()
    M = _rows(x, N, "x")
    if dy.shape != x.shape:
        raise ValueError(f"dy {tuple(dy.shape)} and x {tuple(x.shape)} differ")
    _rows(dy, N, "dy")
    if dy3 is not None and dy2 is None:
        raise ValueError("dy3 needs dy2 (the gradients are summed in order)")
    for name, t in (("dy2", dy2), ("dy3", dy3), ("dres", dres)):
        if t is not None:
            _need(t, name, torch.bfloat16, dev)
            if t.shape != x.shape:
                raise ValueError(f"{name} {tuple(t.shape)} and x {tuple(x.shape)} differ")
            _rows(t, N, name)
    if rstd is not None:
        _need(rstd, "rstd", torch.float32, dev)
        if rstd.numel() != M or not rstd.is_contiguous():
            raise ValueError(f"rstd must be contiguous with {M} elements")
    dx = (torch.empty_like(x) if dx_out is None
          else _check_out(dx_out, "dx_out", torch.bfloat16, dev, shape=x.shape))
    dw = None
    if dw_dtype is not None:
        if dw_dtype not in (torch.float32, torch.bfloat16):
            raise TypeError("dw_dtype must be float32, bfloat16 or None")
        dw = (torch.empty(N, dtype=dw_dtype, device=dev) if dw_out is None
              else _check_out(dw_out, "dw_out", dw_dtype, dev, numel=N))
    with _on_device(dev):
        lib = _lib.load()
        need = int(lib.frag_rmsnorm_bwd_workspace_bytes(M, N))
        if workspace is None or workspace.numel() < need:
            workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
        wc = weight.contiguous()
        tail = (_ptr(x), _ptr(rstd), _ptr(wc), _ptr(dres), _ptr(dx),
                _ptr(dw) if dw_dtype == torch.float32 else None,
                _ptr(dw) if dw_dtype == torch.bfloat16 else None,
                M, N, float(eps), _ptr(workspace), workspace.numel(), _stream(dev))
        if dy3 is None:
            _lib.call("frag_rmsnorm_bwd", _ptr(dy), _ptr(dy2), *tail)
        else:
            _lib.call("frag_rmsnorm_bwd3", _ptr(dy), _ptr(dy2), _ptr(dy3), *tail)
        if return_partials:
            # the launch planned its row blocks from the alignment of every
            # row pointer; ask for the plan of that same case
            aligned = all(t.data_ptr() % 16 == 0
                          for t in (dy, dy2, dy3, x, wc, dres, dx) if t is not None)
            G = int(lib.frag_rmsnorm_bwd_plan_blocks(M, N, int(aligned))) if M else 0
            parts = workspace[: G * N * 4].view(torch.float32).view(G, N)
            return dx, dw, parts
    return dx, dw


def dw_reduce(partials: torch.Tensor, *, out: torch.Tensor | None = None,
              out_bf16: torch.Tensor | None = None) -> torch.Tensor:
    """Fixed-order sum over the rows of a [G, N] fp32 tensor."""
    _need(partials, "partials", torch.float32)
    if partials.dim() != 2 or not partials.is_contiguous():
        raise ValueError("partials must be a contiguous [G, N] tensor")
    G, N = partials.shape
    if out is None and out_bf16 is None:
        out = torch.empty(N, dtype=torch.float32, device=partials.device)
    if out is not None:
        _check_out(out, "out", torch.float32, partials.device, numel=N)
    if out_bf16 is not None:
        _check_out(out_bf16, "out_bf16", torch.bfloat16, partials.device, numel=N)
    with _on_device(partials.device):
        _lib.call("frag_dw_reduce", _ptr(partials), G, N, _ptr(out), _ptr(out_bf16),
                  _stream(partials.device))
    return out if out is not None else out_bf16


# -------------------------------------------------------------- embedding

def embedding_fwd(ids: torch.Tensor, table: torch.Tensor, *, vocab_lo: int = 0,
                  vocab_total: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """out[..., :] = table[ids - vocab_lo] for ids in the shard, zero otherwise.

    table is the whole table (vocab_lo=0) or one contiguous vocab shard
    [vocab_lo, vocab_lo + table.shape[0]) of a vocab_total-row table."""
    _need(ids, "ids", torch.int64)
    _need(table, "table", torch.bfloat16, ids.device)
    if table.dim() != 2 or not table.is_contiguous():
        raise ValueError("table must be a contiguous [rows, D] tensor")
    rows, D = table.shape
    total = rows if vocab_total is None else int(vocab_total)
    ids_c = ids.contiguous()
    T = ids_c.numel()
    o = (torch.empty(*ids.shape, D, dtype=torch.bfloat16, device=ids.device) if out is None
         else _check_out(out, "out", torch.bfloat16, ids.device, shape=(*ids.shape, D)))
    with _on_device(ids.device):
        st = _status_word(ids.device)
        _lib.call("frag_embedding_fwd", _ptr(ids_c), _ptr(table), _ptr(o), T, rows, D,
                  int(vocab_lo), total, _ptr(st), _stream(ids.device))
    if _SYNC_CHECK:
        check_status(ids.device)
    return o


def embedding_rmsnorm_fwd(ids: torch.Tensor, table: torch.Tensor, weight: torch.Tensor,
                          eps: float = 1e-5, *, save_rstd: bool = False,
                          return_embedding: bool = False):
    """y = rmsnorm(table[ids]) * weight without writing the gathered rows to
    HBM (unless return_embedding).  Returns (y, rstd or None, emb or None)."""
    _need(ids, "ids", torch.int64)
    _need(table, "table", torch.bfloat16, ids.device)
    _need(weight, "weight", torch.bfloat16, ids.device)
    if table.dim() != 2 or not table.is_contiguous():
        raise ValueError("table must be a contiguous [rows, D] tensor")
    V, D = table.shape
    if weight.numel() != D:
        raise ValueError(f"weight has {weight.numel()} elements, table rows have {D}")
    ids_c = ids.contiguous()
    T = ids_c.numel()
    y = torch.empty(*ids.shape, D, dtype=torch.bfloat16, device=ids.device)
    rstd = torch.empty(ids.shape, dtype=torch.float32, device=ids.device) if save_rstd else None
    emb = torch.empty_like(y) if return_embedding else None
    wc = weight.contiguous()
    with _on_device(ids.device):
        st = _status_word(ids.device)
        _lib.call("frag_embedding_rmsnorm_fwd", _ptr(ids_c), _ptr(table), _ptr(wc), _ptr(y), _ptr(rstd),
                  _ptr(emb), T, V, D, float(eps), _ptr(st), _stream(ids.device))
    if _SYNC_CHECK:
        check_status(ids.device)
    return y, rstd, emb


def embedding_bwd(grad: torch.Tensor, ids: torch.Tensor, num_rows: int, *, vocab_lo: int = 0,
                  vocab_total: int | None = None, padding_idx: int = -1,
                  out: torch.Tensor | None = None,
                  workspace: torch.Tensor | None = None) -> torch.Tensor:
    """fp32 table gradient G[v] = sum over tokens t (in order) with ids[t] == v of grad[t].

    Every row of G is written (no memset needed).  num_rows is the number of
    table rows this call owns (the whole vocab, or one shard at vocab_lo)."""
    _need(grad, "grad", torch.bfloat16)
    _need(ids, "ids", torch.int64, grad.device)
    D = grad.shape[-1]
    ids_c = ids.contiguous()
    T = ids_c.numel()
    if grad.numel() != T * D:
        raise ValueError(f"grad {tuple(grad.shape)} does not match {T} ids x {D}")
    g = grad.contiguous()
    total = int(num_rows) if vocab_total is None else int(vocab_total)
    G = (torch.empty(num_rows, D, dtype=torch.float32, device=grad.device) if out is None
         else _check_out(out, "out", torch.float32, grad.device, shape=(num_rows, D)))
    with _on_device(grad.device):
        lib = _lib.load()
        need = int(lib.frag_embedding_bwd_workspace_bytes(T, num_rows))
        if need == 0 and num_rows > 0:
            raise FragError("frag_embedding_bwd_workspace_bytes", 2, "unsupported sizes")
        if workspace is None or workspace.numel() < need:
            workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=grad.device)
        st = _status_word(grad.device)
        _lib.call("frag_embedding_bwd", _ptr(ids_c), _ptr(g), _ptr(G), T, int(num_rows), D,
                  int(vocab_lo), total, int(padding_idx), _ptr(workspace), workspace.numel(),
                  _ptr(st), _stream(grad.device))
    if _SYNC_CHECK:
        check_status(grad.device)
    return G


def rmsnorm_embedding_bwd(x: torch.Tensor, weight: torch.Tensor, ids: torch.Tensor,
                          dy: torch.Tensor | tuple | list, num_rows: int, *,
                          rstd: torch.Tensor | None = None, dres: torch.Tensor | None = None,
                          eps: float = 1e-5, write_y: bool = False, return_d_emb: bool = False,
                          dw_dtype: torch.dtype = torch.float32, vocab_lo: int = 0,
                          vocab_total: int | None = None, padding_idx: int = -1,
                          out: torch.Tensor | None = None,
                          workspace: torch.Tensor | None = None):
    """RMSNorm backward fused into the table-gradient scatter of its input
    gradient (the first attention_norm after the token embedding).

    x      the embedding output that entered the norm, bf16 [..., D]
    dy     one bf16 gradient, or a sequence of up to three summed in order in
           bf16 (bf16(bf16(a + b) + c), as the reference graph adds them)
    rstd   saved rstd (fp32, one per token) or None to recompute it with eps
    dres   optional residual gradient added (bf16) to the norm's dx
    Returns (G fp32 [num_rows, D], dw [D] (fp32 or bf16), y or None, d_emb or None):
    y is the recomputed forward bf16(x * rstd * w) (write_y), d_emb the
    gradient the scatter consumed (return_d_emb; otherwise never stored)."""
    terms = list(dy) if isinstance(dy, (tuple, list)) else [dy]
    if not 1 <= len(terms) <= 3:
        raise ValueError("dy must be one tensor or a sequence of one to three tensors")
    _need(x, "x", torch.bfloat16)
    dev = x.device
    _need(weight, "weight", torch.bfloat16, dev)
    _need(ids, "ids", torch.int64, dev)
    D = weight.numel()
    T = _rows(x, D, "x")
    if ids.numel() != T:
        raise ValueError(f"ids has {ids.numel()} elements, x has {T} rows")
    for j, t in enumerate(terms):
        _need(t, f"dy[{j}]", torch.bfloat16, dev)
        if t.numel() != x.numel():
            raise ValueError(f"dy[{j}] {tuple(t.shape)} does not match x {tuple(x.shape)}")
        _rows(t, D, f"dy[{j}]")
    if dres is not None:
        _need(dres, "dres", torch.bfloat16, dev)
        if dres.numel() != x.numel():
            raise ValueError(f"dres {tuple(dres.shape)} does not match x {tuple(x.shape)}")
        _rows(dres, D, "dres")
    if rstd is not None:
        _need(rstd, "rstd", torch.float32, dev)
        if rstd.numel() != T or not rstd.is_contiguous():
            raise ValueError(f"rstd must be contiguous with {T} elements")
    if dw_dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("dw_dtype must be float32 or bfloat16")
    ids_c = ids.contiguous()
    total = int(num_rows) if vocab_total is None else int(vocab_total)
    G = (torch.empty(num_rows, D, dtype=torch.float32, device=dev) if out is None
         else _check_out(out, "out", torch.float32, dev, shape=(num_rows, D)))
    dw = torch.empty(D, dtype=dw_dtype, device=dev)
    y = torch.empty_like(x) if write_y else None
    d_emb = torch.empty_like(x) if return_d_emb else None
    a, b, c = (terms + [None, None])[:3]
    wc = weight.contiguous()
    with _on_device(dev):
        lib = _lib.load()
        need = int(lib.frag_rmsnorm_embedding_bwd_workspace_bytes(T, D, num_rows))
        if need == 0 and D > 0:
            raise FragError("frag_rmsnorm_embedding_bwd_workspace_bytes", 2, "unsupported sizes")
        if workspace is None or workspace.numel() < need:
            workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
        st = _status_word(dev)
        _lib.call("frag_rmsnorm_embedding_bwd", _ptr(x), _ptr(wc), _ptr(rstd), _ptr(y),
                  _ptr(a), _ptr(b), _ptr(c), _ptr(dres), _ptr(d_emb), _ptr(ids_c), _ptr(G),
                  _ptr(dw) if dw_dtype == torch.float32 else None,
                  _ptr(dw) if dw_dtype == torch.bfloat16 else None,
                  T, D, int(num_rows), int(vocab_lo), total, int(padding_idx), float(eps),
                  _ptr(workspace), workspace.numel(), _ptr(st), _stream(dev))
    if _SYNC_CHECK:
        check_status(dev)
    return G, dw, y, d_emb


def copy_rows(src: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Contiguous copy of a 2-D tensor whose rows are contiguous but may be
    strided apart (a split of an FSDP all-gather buffer viewed [world, -1]).
    Returns a new [rows, cols] tensor (or fills `out`)."""
    _check_copy_src(src)
    rows, cols = src.shape
    if out is None:
        out = torch.empty(rows, cols, dtype=src.dtype, device=src.device)
    elif out.shape != src.shape or out.dtype != src.dtype or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of src's shape and dtype")
    es = src.element_size()
    with _on_device(src.device):
        _lib.call("frag_copy_rows", _ptr(src), src.stride(0) * es, _ptr(out), cols * es, rows,
                  cols * es, _stream(src.device))
    return out


def _check_copy_src(src: torch.Tensor) -> None:
    if not isinstance(src, torch.Tensor):
        raise TypeError("src must be a torch.Tensor")
    if not src.is_cuda:
        raise ValueError("src must be a CUDA tensor")
    if src.dim() != 2 or (src.shape[1] > 1 and src.stride(1) != 1):
        raise ValueError("src must be 2-D with contiguous rows")


def copy_rows_grouped(srcs, outs=None) -> list[torch.Tensor]:
    """copy_rows for up to 16 sources in one launch (frag_copy_rows_grouped):
    the splits of one FSDP all-gather buffer viewed [world, -1].  Returns the
    contiguous copies in order (or fills the given `outs`, None entries
    allocated)."""
    srcs = list(srcs)
    if len(srcs) > _lib.FRAG_COPY_MAX_SEGMENTS:
        raise ValueError(f"at most {_lib.FRAG_COPY_MAX_SEGMENTS} sources per group")
    outs = [None] * len(srcs) if outs is None else list(outs)
    if len(outs) != len(srcs):
        raise ValueError("outs must match srcs in length")
    if not srcs:
        return []
    for src in srcs:
        _check_copy_src(src)
    dev = srcs[0].device
    if any(src.device != dev for src in srcs):
        raise ValueError("all sources must be on one device")
    segs = (_lib.CopySegment * len(srcs))()
    for i, src in enumerate(srcs):
        rows, cols = src.shape
        out = outs[i]
        if out is None:
            out = outs[i] = torch.empty(rows, cols, dtype=src.dtype, device=dev)
        elif (out.shape != src.shape or out.dtype != src.dtype or not out.is_contiguous()
              or out.device != dev):
            raise ValueError("each out must be a contiguous tensor of its src's shape and dtype")
        es = src.element_size()
        segs[i] = _lib.CopySegment(src.data_ptr(), out.data_ptr(), src.stride(0) * es, cols * es,
                                   rows, cols * es)
    with _on_device(dev):
        _lib.call("frag_copy_rows_grouped", segs, len(srcs), _stream(dev))
    return outs


_DT = {torch.bfloat16: _lib.FRAG_DT_BF16, torch.float32: _lib.FRAG_DT_F32}


def convert(src: torch.Tensor, dtype: torch.dtype, copies: int = 1):
    """bf16 <-> fp32 element type conversion (frag_convert_rows): a new
    contiguous tensor of src's shape in `dtype` (fp32 -> bf16 rounds to
    nearest even), or a tuple of `copies` (1 or 2) such tensors written by
    one pass.  src may be any view whose last dimension is contiguous and
    whose leading dimensions collapse into one row stride."""
    if not isinstance(src, torch.Tensor) or src.dtype not in _DT or dtype not in _DT:
        raise TypeError("convert takes bfloat16 / float32 tensors and dtypes")
    if not src.is_cuda:
        raise ValueError("src must be a CUDA tensor")
    if copies not in (1, 2):
        raise ValueError("copies must be 1 or 2")
    cols = src.shape[-1] if src.dim() else 1
    try:
        rows2d = src.view(-1, cols) if src.dim() else src.view(1, 1)
    except RuntimeError:
        raise ValueError("src's leading dimensions must collapse into one row stride") from None
    if cols > 1 and rows2d.stride(1) != 1:
        raise ValueError("src's last dimension must be contiguous")
    outs = [torch.empty(src.shape, dtype=dtype, device=src.device) for _ in range(copies)]
    rows = rows2d.shape[0]
    with _on_device(src.device):
        _lib.call("frag_convert_rows", _ptr(rows2d), _DT[src.dtype], rows2d.stride(0) if rows > 1 else cols,
                  _ptr(outs[0]), _ptr(outs[1]) if copies == 2 else None, _DT[dtype], cols, rows, cols,
                  _stream(src.device))
    return outs[0] if copies == 1 else tuple(outs)


# ------------------------------------------------------------------- RoPE

_LAYOUTS = {"neox": _lib.FRAG_ROPE_NEOX, "interleaved": _lib.FRAG_ROPE_INTERLEAVED}


def _rope_desc(x: torch.Tensor, out: torch.Tensor, name: str) -> _lib.RopeTensor:
    if x.dim() != 4:
        raise ValueError(f"{name} must be [B, S, H, D] (any strides, last dim contiguous)")
    if x.stride(-1) != 1 or out.stride(-1) != 1:
        raise ValueError(f"{name}: the head dimension must be contiguous")
    if out.shape != x.shape:
        raise ValueError(f"{name}: output shape {tuple(out.shape)} != {tuple(x.shape)}")
    if out.dtype not in (torch.bfloat16, torch.float32) or out.device != x.device:
        raise TypeError(f"{name}: the output must be bf16 or float32 on {x.device}")
    B, S, H, D = x.shape
    odt = _lib.FRAG_ROPE_OUT_F32 if out.dtype == torch.float32 else _lib.FRAG_ROPE_OUT_BF16
    idt = _lib.FRAG_ROPE_IN_F32 if x.dtype == torch.float32 else _lib.FRAG_ROPE_IN_BF16
    if idt == _lib.FRAG_ROPE_IN_F32 and odt != _lib.FRAG_ROPE_OUT_F32:
        raise TypeError(f"{name}: a float32 input needs a float32 output")
    return _lib.RopeTensor(x.data_ptr(), out.data_ptr(), H, x.stride(0), x.stride(1), x.stride(2),
                           out.stride(0), out.stride(1), out.stride(2), odt, idt)


def rope_complex(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor | None,
                 freqs: torch.Tensor, *, inverse: bool = False, out_q: torch.Tensor | None = None,
                 out_k: torch.Tensor | None = None):
    """The complex multiply of the v1/v2 snapshots: q (and k) complex64
    [B, S, H, D/2] times freqs[positions] (complex64 [P, D/2]; positions None
    = s), complex64 results (new, or the given out_q / out_k), fp32
    arithmetic throughout -> (out_q, out_k)."""
    def real(t, name):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.complex64 or t.dim() != 4:
            raise TypeError(f"{name} must be a complex64 [B, S, H, D/2] tensor")
        if t.stride(-1) != 1:
            raise ValueError(f"{name}: the last dimension must be contiguous")
        return torch.view_as_real(t).flatten(-2)
    oq = torch.empty(q.shape, dtype=torch.complex64, device=q.device) if out_q is None else out_q
    ok = None
    if k is not None:
        ok = torch.empty(k.shape, dtype=torch.complex64, device=k.device) if out_k is None else out_k
    rope(real(q, "q"), None if k is None else real(k, "k"), positions, theta=None, freqs=freqs,
         layout="interleaved", inverse=inverse, out_q=real(oq, "out_q"),
         out_k=None if ok is None else real(ok, "out_k"))
    return oq, ok


def _new_out(x: torch.Tensor, out_layout: str) -> torch.Tensor:
    B, S, H, D = x.shape
    if out_layout == "bshd":
        return torch.empty((B, S, H, D), dtype=x.dtype, device=x.device)
    if out_layout == "bhsd":  # [B, H, S, D] storage, returned as a [B, S, H, D] view
        return torch.empty((B, H, S, D), dtype=x.dtype, device=x.device).transpose(1, 2)
    raise ValueError("out_layout must be 'bshd' or 'bhsd'")


def rope(q: torch.Tensor, k: torch.Tensor | None = None, positions: torch.Tensor | None = None, *,
         theta: float | None = 500000.0, freqs: torch.Tensor | None = None,
         layout: str = "neox", inverse: bool = False, out_q: torch.Tensor | None = None,
         out_k: torch.Tensor | None = None, out_layout: str = "bshd"):
    """Rotary embedding of q (and k) given as [B, S, H, D] views (any strides,
    contiguous head dim).  Returns (out_q, out_k); outputs default to new
    contiguous tensors and may alias the inputs (in-place).

    positions: int32/int64 [B, S] (or [S], broadcast over B), or None for
    position = s.  freqs: complex64 [P, D/2] table indexed by position (the
    reference's freqs_cis input); without it cos/sin are computed in
    registers from theta.  inverse=True applies the conjugate rotation (the
    backward).  out_layout="bhsd" writes new outputs in the [B, H, S, D]
    storage order attention kernels read (the transpose is fused into the
    stores; the returned tensors are [B, S, H, D] views of that storage, so
    `.transpose(1, 2)` gives contiguous [B, H, S, D]).  An out_q / out_k of
    dtype float32 receives the rotated values unrounded.  float32 q and k
    (complex64 tensors viewed as (re, im) pairs, see rope_complex) take the
    interleaved layout and float32 outputs."""
    if not isinstance(q, torch.Tensor) or q.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("q must be a bfloat16 or float32 torch.Tensor")
    if not q.is_cuda:
        raise ValueError("q must be a CUDA tensor")
    dev = q.device
    if q.dtype == torch.float32 and layout != "interleaved":
        raise ValueError("float32 (complex) inputs take the interleaved layout")
    if layout not in _LAYOUTS:
        raise ValueError(f"layout must be one of {sorted(_LAYOUTS)}")
    B, S, Hq, D = q.shape
    oq = _new_out(q, out_layout) if out_q is None else out_q
    descs = [_rope_desc(q, oq, "q")]
    ok = None
    if k is not None:
        _need(k, "k", q.dtype, dev)
        if k.shape[0] != B or k.shape[1] != S or k.shape[3] != D:
            raise ValueError(f"k {tuple(k.shape)} does not match q {tuple(q.shape)}")
        ok = _new_out(k, out_layout) if out_k is None else out_k
        descs.append(_rope_desc(k, ok, "k"))
    arr = (_lib.RopeTensor * len(descs))(*descs)
    pos_ptr, pos_dtype, psb, pss = None, _lib.FRAG_POS_NONE, 0, 0
    if positions is not None:
        if positions.device != dev:
            raise ValueError("positions must be on the same device as q")
        if positions.dtype == torch.int64:
            pos_dtype = _lib.FRAG_POS_I64
        elif positions.dtype == torch.int32:
            pos_dtype = _lib.FRAG_POS_I32
        else:
            raise TypeError("positions must be int32 or int64")
        if positions.dim() == 1:
            if positions.shape[0] != S:
                raise ValueError("1-D positions must have S entries")
            psb, pss = 0, positions.stride(0)
        elif positions.dim() == 2 and tuple(positions.shape) == (B, S):
            psb, pss = positions.stride(0), positions.stride(1)
        else:
            raise ValueError(f"positions must be [B, S] or [S], got {tuple(positions.shape)}")
        pos_ptr = C.c_void_p(positions.data_ptr())
    fptr, fstride, frows = None, 0, 0
    if freqs is not None:
        if freqs.dtype != torch.complex64 or freqs.device != dev:
            raise TypeError("freqs must be a complex64 tensor on q's device")
        f2 = freqs.reshape(-1, freqs.shape[-1])
        if f2.shape[-1] != D // 2 or f2.stride(-1) != 1:
            raise ValueError(f"freqs rows must hold D/2={D // 2} contiguous complex values")
        fptr, fstride, frows = C.c_void_p(f2.data_ptr()), f2.stride(0), f2.shape[0]
        theta_v = 0.0
    else:
        if theta is None:
            raise ValueError("either theta or freqs is required")
        theta_v = float(theta)
    with _on_device(dev):
        _lib.call("frag_rope", arr, len(descs), B, S, D, pos_ptr, pos_dtype, psb, pss, fptr,
                  fstride, frows, theta_v, _LAYOUTS[layout], int(bool(inverse)), _stream(dev))
    return oq, ok


class RopeFrequencies:
    """The frequencies of a rotary embedding, computed once in 64 bits and kept
    on the host: pass it to rope_scaled.

    head_dim       elements of a head; rotary_dim (default all) of them, the
                   first, are rotated, the others pass through
    theta          base: pair j turns by theta^(-2j / rotary_dim) a position
    scaling        how the frequencies f are slowed for contexts `factor` times
                   original_context long:
      "none"       not at all
      "linear"     f / factor (positions are interpolated)
      "base"       theta * factor^(rotary_dim / (rotary_dim - 2)): the last
                   pair is slowed by the factor, the first not at all
      "smooth"     by the turns a pair makes in original_context: fewer than
                   low_turns f / factor, more than high_turns f, between them
                   a linear blend
      "parts"      a blend linear in the pair's index, f up to the pair that
                   makes fast_turns in original_context, f / factor from the
                   one that makes slow_turns; rotated values are multiplied by
                   0.1 ln(factor) + 1
    attention_factor  replaces that multiplier (1 for the other scalings)

    `turns` (float64 tensor [rotary_dim / 2]) holds f / (2 pi)."""

    def __init__(self, head_dim: int, *, rotary_dim: int | None = None, theta: float = 500000.0,
                 scaling: str = "none", factor: float = 1.0, original_context: int = 8192,
                 low_turns: float = 1.0, high_turns: float = 4.0, fast_turns: float = 32.0,
                 slow_turns: float = 1.0, attention_factor: float | None = None):
        rot = head_dim if rotary_dim is None else rotary_dim
        if rot <= 0 or rot % 2 or rot > head_dim:
            raise ValueError(f"rotary_dim must be even and in (0, {head_dim}], got {rot}")
        if rot > 512:
            raise ValueError(f"rotary_dim must be at most 512, got {rot}")
        if not theta > 1 or not math.isfinite(theta):
            raise ValueError("theta must be finite and above 1")
        if scaling not in ("none", "linear", "base", "smooth", "parts"):
            raise ValueError(f"unknown scaling {scaling!r}")
        if not factor >= 1 or not math.isfinite(factor):
            raise ValueError("factor must be finite and at least 1")
        if original_context <= 0:
            raise ValueError("original_context must be positive")
        if not high_turns > low_turns > 0 or not fast_turns > slow_turns > 0:
            raise ValueError("high_turns must be above low_turns, and fast_turns above slow_turns, all positive")
        self.head_dim, self.rotary_dim = head_dim, rot
        if scaling == "base":
            if rot < 4:
                raise ValueError("scaling 'base' needs a rotary_dim of at least 4")
            theta = theta * factor ** (rot / (rot - 2))
        j = torch.arange(rot // 2, dtype=torch.float64)
        turns = theta ** (-2.0 * j / rot) / (2 * math.pi)
        self.attention_factor = 1.0
        if scaling == "linear":
            turns = turns / factor
        elif scaling == "smooth":
            keep = ((turns * original_context - low_turns) / (high_turns - low_turns)).clamp(0, 1)
            turns = turns * (keep + (1 - keep) / factor)
        elif scaling == "parts":
            def pair(n):  # the (fractional) pair that makes n turns in the original context
                return rot * math.log(original_context / (2 * math.pi * n)) / (2 * math.log(theta))
            first, last = max(math.floor(pair(fast_turns)), 0), min(math.ceil(pair(slow_turns)), rot - 1)
            slowed = ((j - first) / max(last - first, 1e-3)).clamp(0, 1)
            turns = turns * (1 - slowed + slowed / factor)
            self.attention_factor = 0.1 * math.log(factor) + 1.0
        if attention_factor is not None:
            self.attention_factor = float(attention_factor)
        self.turns = turns
        self._turns = (C.c_double * (rot // 2))(*turns.tolist())


def _overlaps(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors share memory.  Where their address ranges meet, as
    those of head slices of one packed tensor do, the strides decide: an element
    of each has the same address where sum(stride * index difference) is the
    distance of the two, with the index differences of equal strides taken
    together.  The largest stride goes first, and as soon as the strides left
    reach every distance within their span the question is answered."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    distance = b.data_ptr() - a.data_ptr()
    reach = {1: [1 - b.element_size(), a.element_size() - 1]}  # stride in bytes: index differences
    for t, at in ((b, 0), (a, 1)):
        for n, s in zip(t.shape, t.stride()):
            if n > 1 and s > 0:
                r = reach.setdefault(s * t.element_size(), [0, 0])
                r[at] += n - 1 if at else 1 - n
    strides = sorted(reach, reverse=True)
    lo, hi = [0], [0]  # of the strides from i on
    dense = [True]
    for s in reversed(strides):
        dense.insert(0, dense[0] and s <= hi[0] - lo[0] + 1)
        lo.insert(0, lo[0] + s * reach[s][0])
        hi.insert(0, hi[0] + s * reach[s][1])
    left = [4096]  # cases to look at; what is not settled by then counts as shared

    def meet(i: int, d: int) -> bool:
        if not lo[i] <= d <= hi[i]:
            return False
        if dense[i]:
            return True
        s = strides[i]
        for k in range(max(reach[s][0], -((hi[i + 1] - d) // s)), min(reach[s][1], (d - lo[i + 1]) // s) + 1):
            left[0] -= 1
            if left[0] < 0 or meet(i + 1, d - k * s):
                return True
        return False
    return meet(0, distance)


def _check_rope_out(x: torch.Tensor, out: torch.Tensor, name: str) -> None:
    if not isinstance(out, torch.Tensor) or out.dtype != torch.bfloat16 or out.device != x.device:
        raise TypeError(f"{name}: the output must be a bfloat16 tensor on {x.device}")
    if out.shape != x.shape:
        raise ValueError(f"{name}: output shape {tuple(out.shape)} != {tuple(x.shape)}")
    if any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
        raise ValueError(f"{name}: the output must not repeat elements (an expanded view)")
    same = out.data_ptr() == x.data_ptr() and all(
        n <= 1 or a == b for n, a, b in zip(x.shape, x.stride(), out.stride()))
    if not same and _overlaps(x, out):
        raise ValueError(f"{name}: the output overlaps the input without being the same view")


def _check_rope_outs(q: torch.Tensor, k: torch.Tensor, oq: torch.Tensor, ok: torch.Tensor) -> None:
    """One launch reads q and k while it writes the outputs, heads of a token
    by different warps: neither output may share memory with the other input or
    the other output.  (In place the three questions are one.)"""
    if _overlaps(oq, ok):
        raise ValueError("out_q and out_k overlap")
    if ok is not k and _overlaps(oq, k):
        raise ValueError("out_q overlaps k")
    if oq is not q and _overlaps(ok, q):
        raise ValueError("out_k overlaps q")


def rope_scaled(q: torch.Tensor, k: torch.Tensor | None = None, positions: torch.Tensor | None = None, *,
                freqs: RopeFrequencies, layout: str = "neox", backward: bool = False,
                out_q: torch.Tensor | None = None, out_k: torch.Tensor | None = None,
                out_layout: str = "bshd"):
    """Rotary embedding of bf16 q (and k), [B, S, H, D] views of any strides
    with a contiguous head dimension, by a RopeFrequencies plan: the first
    freqs.rotary_dim elements of every head are rotated (pairs (j, j +
    rotary_dim/2) for layout "neox", (2j, 2j+1) for "interleaved"), the others
    pass through.  Returns (out_q, out_k), new contiguous tensors or the given
    out_q / out_k, which may be q and k themselves (in place); an output must not
    share memory with its input in any other way, nor with the other input or
    output (slices of one packed tensor, in either order of heads and tokens,
    are fine).

    positions: int32/int64 [B, S] or [S], or None for position = s.  A product
    of position and frequency is taken in 64 bits, so a long context's last
    token is as exact as its first; rotated values are rounded once.
    backward=True gives the gradient: the transposed rotation, with the same
    attention factor.  out_layout as in rope."""
    _need(q, "q", torch.bfloat16)
    dev = q.device
    if not isinstance(freqs, RopeFrequencies):
        raise TypeError("freqs must be a RopeFrequencies")
    if layout not in _LAYOUTS:
        raise ValueError(f"layout must be one of {sorted(_LAYOUTS)}")
    if q.dim() != 4:
        raise ValueError("q must be [B, S, H, D] (any strides, last dim contiguous)")
    B, S, _, D = q.shape
    if D != freqs.head_dim:
        raise ValueError(f"q has heads of {D} elements, the plan is for {freqs.head_dim}")
    oq, dq = _rope_pair(q, out_q, out_layout, "q")
    ok = None
    if k is None:
        arr = (_lib.RopeTensor * 1)(dq)
    else:
        _need(k, "k", torch.bfloat16, dev)
        if k.dim() != 4 or k.shape[0] != B or k.shape[1] != S or k.shape[3] != D:
            raise ValueError(f"k {tuple(k.shape)} does not match q {tuple(q.shape)}")
        ok, dk = _rope_pair(k, out_k, out_layout, "k")
        if out_q is not None or out_k is not None:
            _check_rope_outs(q, k, oq, ok)
        arr = (_lib.RopeTensor * 2)(dq, dk)
    pos_ptr, pos_dtype, psb, pss = _rope_positions(positions, B, S, dev)
    with _on_device(dev):
        _lib.call("frag_rope_scaled", arr, 1 if k is None else 2, B, S, D, freqs.rotary_dim, pos_ptr, pos_dtype, psb,
                  pss, freqs._turns, freqs.attention_factor, _LAYOUTS[layout], 1 if backward else 0, _stream(dev))
    return oq, ok


def _rope_pair(x: torch.Tensor, out: torch.Tensor | None, out_layout: str, name: str):
    """x's output, checked or new, and the descriptor of the two."""
    if x.stride(-1) != 1:
        raise ValueError(f"{name}: the head dimension must be contiguous")
    if out is not None:
        _check_rope_out(x, out, name)
        if out.stride(-1) != 1:
            raise ValueError(f"{name}: the output's head dimension must be contiguous")
    elif out_layout == "bshd":
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    else:
        out = _new_out(x, out_layout)
    xs, os_ = x.stride(), out.stride()
    return out, _lib.RopeTensor(x.data_ptr(), out.data_ptr(), x.shape[2], xs[0], xs[1], xs[2], os_[0], os_[1], os_[2],
                                _lib.FRAG_ROPE_OUT_BF16, _lib.FRAG_ROPE_IN_BF16)


def _rope_positions(positions, B: int, S: int, dev: torch.device):
    """(pointer, dtype code, batch stride, sequence stride) of a position tensor."""
    if positions is None:
        return None, _lib.FRAG_POS_NONE, 0, 0
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
        raise TypeError("positions must be an int32 or int64 tensor")
    if positions.device != dev:
        raise ValueError("positions must be on the same device as q")
    code = _lib.FRAG_POS_I64 if positions.dtype == torch.int64 else _lib.FRAG_POS_I32
    if positions.dim() == 1 and positions.shape[0] == S:
        return positions.data_ptr(), code, 0, positions.stride(0)
    if positions.dim() == 2 and tuple(positions.shape) == (B, S):
        return positions.data_ptr(), code, positions.stride(0), positions.stride(1)
    raise ValueError(f"positions must be [B, S] or [S], got {tuple(positions.shape)}")


# ------------------------------------------------- RMSNorm in 8 bits and scales

_FP8 = {torch.float8_e4m3fn: _lib.FRAG_FP8_E4M3, torch.float8_e5m2: _lib.FRAG_FP8_E5M2}
_GROUPS = (0, 32, 64, 128)


def _strided_rows(t: torch.Tensor, name: str, N: int, dev: torch.device, shape=None,
                  dtype: torch.dtype = torch.bfloat16):
    """(the tensor, row stride) of a tensor whose rows of N are
    contiguous and whose leading dimensions collapse into one row stride."""
    _need(t, name, dtype, dev)
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} {tuple(t.shape)} and x {tuple(shape)} differ")
    if t.dim() < 1 or t.shape[-1] != N:
        raise ValueError(f"{name}: last dim of {tuple(t.shape)} != normalized size {N}")
    if t.is_contiguous():
        return t, N
    try:
        rows = t.view(-1, N) if t.numel() else t
    except RuntimeError:
        raise ValueError(f"{name}'s leading dimensions must collapse into one row stride") from None
    if N > 1 and rows.stride(-1) != 1:
        raise ValueError(f"{name}'s rows must be contiguous")
    return rows, rows.stride(0) if rows.dim() == 2 else N


def _width(weight: torch.Tensor, x: torch.Tensor) -> int:
    """Values of a row.  Rows of none have no mean: refused, as by the C entry."""
    N = weight.numel()
    if N == 0 and math.prod(x.shape[:-1]):
        raise ValueError("rows must hold at least one value")
    return N


def _quant_out(x: torch.Tensor, N: int, dtype, group: int, scale_dtype, dev):
    if dtype not in _FP8:
        raise TypeError("dtype must be float8_e4m3fn or float8_e5m2")
    if group not in _GROUPS:
        raise ValueError(f"group must be one of {_GROUPS} (0: one scale for a row)")
    if scale_dtype not in (torch.float32, torch.float8_e8m0fnu):
        raise TypeError("scale_dtype must be float32 or float8_e8m0fnu")
    q = torch.empty_like(x, dtype=dtype, memory_format=torch.contiguous_format)
    shape = x.shape[:-1] + (-(-N // group),) if group else x.shape[:-1]
    return q, _new(x, shape, scale_dtype)


def _workspace(given: torch.Tensor | None, need: int, like: torch.Tensor):
    """(pointer, bytes, the tensor) of the caller's workspace where it is large
    enough, or of a new one; nothing where none is needed."""
    if given is not None:
        if not isinstance(given, torch.Tensor) or given.device != like.device or not given.is_contiguous():
            raise ValueError(f"workspace must be a contiguous tensor on {like.device}")
        if need and given.numel() * given.element_size() >= need and given.data_ptr() % 256 == 0:
            return given.data_ptr(), given.numel() * given.element_size(), given
    if need == 0:
        return None, 0, None
    new = like.new_empty(need, dtype=torch.uint8)
    return new.data_ptr(), need, new


def rmsnorm_quant_fwd(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, *,
                      residual: torch.Tensor | None = None, dtype: torch.dtype = torch.float8_e4m3fn,
                      group: int = 0, scale_dtype: torch.dtype = torch.float32, write_h: bool = True,
                      save_rstd: bool = True):
    """(Residual add +) RMSNorm with its output in 8 bits and scales, in one
    pass.  Returns (q, scale, h, rstd): y = rmsnorm(h) * w is q * scale.

    h      bf16(residual + x): the new residual stream, which the backward
           (rmsnorm_quant_bwd, rmsnorm_bwd) takes as its x; None without a
           residual or with write_h=False
    q      float8_e4m3fn or float8_e5m2, shaped like x, rounded from 32 bits
    scale  max |y| / the format's largest value, for each row (group=0, shaped
           x.shape[:-1]) or each `group` of its values (x.shape[:-1] +
           [ceil(N / group)], the last one of a row may be cut); 1 where all
           are zero.  scale_dtype=float8_e8m0fnu rounds it up to a power of two
    rstd   fp32 x.shape[:-1], or None

    x and residual: rows of weight.numel() contiguous values, any row stride."""
    _need(x, "x", torch.bfloat16)
    dev = x.device
    _need(weight, "weight", torch.bfloat16, dev)
    N = _width(weight, x)
    x2, xs = _strided_rows(x, "x", N, dev)
    r2, rs = (None, 0) if residual is None else _strided_rows(residual, "residual", N, dev, x.shape)
    q, scale = _quant_out(x, N, dtype, group, scale_dtype, dev)
    h = None
    if residual is not None and write_h:
        h = torch.empty_like(x, memory_format=torch.contiguous_format)
    rstd = _new(x, x.shape[:-1], torch.float32) if save_rstd else None
    wc = weight.contiguous()
    with _on_device(dev):
        _lib.call("frag_rmsnorm_quant_fwd", _ptr(x2), xs, _ptr(r2), rs, _ptr(wc), _ptr(q), _ptr(scale), _ptr(h),
                  _ptr(rstd), x.numel() // N if N else 0, N, float(eps), _FP8[dtype], group,
                  int(scale_dtype != torch.float32), _stream(dev))
    return q, scale, h, rstd


def rmsnorm_quant_bwd(dy: torch.Tensor, x: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor, *,
                      dres: torch.Tensor | None = None, dtype: torch.dtype = torch.float8_e5m2, group: int = 0,
                      scale_dtype: torch.dtype = torch.float32, write_dx: bool = True, compute_dw: bool = True,
                      workspace: torch.Tensor | None = None):
    """The gradient of (residual add +) RMSNorm in bf16 and, for the
    projection below the residual, in 8 bits and scales, in one pass.
    Returns (dx, q, scale, dw).

    dy     gradient of the norm's output (the 8-bit rounding passes it through)
    x      the normalised input (h of rmsnorm_quant_fwd), rstd its saved fp32
    dres   the residual stream's own gradient, added to dx
    dx     bf16(dres + RMSNorm backward), rounded once, or None; q and scale
           are of the same 32-bit values, as in rmsnorm_quant_fwd
    dw     fp32 [N] summed in a fixed order, or None"""
    _need(x, "x", torch.bfloat16)
    dev = x.device
    _need(weight, "weight", torch.bfloat16, dev)
    N = _width(weight, x)
    x2, xs = _strided_rows(x, "x", N, dev)
    y2, ys = _strided_rows(dy, "dy", N, dev, x.shape)
    r2, rs = (None, 0) if dres is None else _strided_rows(dres, "dres", N, dev, x.shape)
    M = x.numel() // N if N else 0
    _need(rstd, "rstd", torch.float32, dev)
    if rstd.numel() != M or not rstd.is_contiguous():
        raise ValueError(f"rstd must be contiguous with {M} elements")
    q, scale = _quant_out(x, N, dtype, group, scale_dtype, dev)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if write_dx else None
    dw = weight.new_empty(N, dtype=torch.float32) if compute_dw else None
    wc = weight.contiguous()
    with _on_device(dev):
        need = int(_lib.load().frag_rmsnorm_quant_bwd_workspace_bytes(M, N))
        ws, ws_bytes, workspace = _workspace(workspace, need, x)
        _lib.call("frag_rmsnorm_quant_bwd", _ptr(y2), ys, _ptr(x2), xs, _ptr(rstd), _ptr(wc), _ptr(r2), rs,
                  _ptr(dx), _ptr(q), _ptr(scale), _ptr(dw), M, N, _FP8[dtype], group,
                  int(scale_dtype != torch.float32), ws, ws_bytes, _stream(dev))
    return dx, q, scale, dw


# --------------------------------------------- orthogonalised weight updates

NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)


def _matrices(t: torch.Tensor, name: str, dev: torch.device | None = None, shape=None):
    """(E, m, n, descriptor) of a bf16 or fp32 [..., m, n] tensor whose
    leading dimensions collapse into one stride."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in _DT:
        raise TypeError(f"{name} must be bfloat16 or float32, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if dev is not None and t.device != dev:
        raise ValueError(f"{name} is on {t.device}, expected {dev}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} {tuple(t.shape)} != {tuple(shape)}")
    if t.dim() < 2:
        raise ValueError(f"{name} must be [..., m, n], got {tuple(t.shape)}")
    m, n = t.shape[-2:]
    E = 1
    for d in t.shape[:-2]:
        E *= d
    sb = span = None
    if E > 0:  # one stride for the leading dimensions together
        for size, stride in zip(reversed(t.shape[:-2]), reversed(t.stride()[:-2])):
            if size == 1:
                continue
            if sb is None:
                sb, span = stride, size * stride
            elif stride != span:
                raise ValueError(f"{name}'s leading dimensions must collapse into one stride")
            else:
                span *= size
    return E, m, n, _lib.Matrix(t.data_ptr(), sb or 0, t.stride(-2), t.stride(-1), _DT[t.dtype])


def _check_replaces(out: torch.Tensor, name: str, like: torch.Tensor, inputs) -> None:
    """A contiguous output may be `like` itself, element by element.  Any other
    memory shared with an input is refused: a stack's matrices are not written
    in the order in which they are read."""
    for t in inputs:
        if _overlaps(out, t) and not (t is like and out.data_ptr() == t.data_ptr() and t.is_contiguous()
                                      and out.dtype == t.dtype):
            raise ValueError(f"{name} overlaps an input that it does not replace")


@functools.lru_cache(maxsize=64)
def _repeated(steps: int, a: float, b: float, c: float):
    return (C.c_float * (3 * steps))(*([a, b, c] * steps))


def _schedule(steps: int, coefficients):
    """The C array of `steps` triples: one triple for all, or one for each."""
    if not isinstance(steps, int) or not 1 <= steps <= 32:
        raise ValueError("steps must be an integer from 1 to 32")
    rows = list(coefficients)
    if len(rows) == 3 and all(isinstance(c, (int, float)) for c in rows):
        if not all(math.isfinite(c) for c in rows):
            raise ValueError("coefficients must be finite")
        return _repeated(steps, *rows)
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        raise ValueError("coefficients must be a triple (a, b, c) or one for each step")
    flat = [float(c) for r in rows for c in r]
    if not all(math.isfinite(c) for c in flat):
        raise ValueError("coefficients must be finite")
    return (C.c_float * len(flat))(*flat)


def orthogonalize_workspace_bytes(E: int, m: int, n: int) -> int:
    return int(_lib.load().frag_orthogonalize_workspace_bytes(E, m, n))


def orthogonalize(g: torch.Tensor, *, steps: int = 5, coefficients=NEWTON_SCHULZ, eps: float = 1e-7,
                  out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Newton-Schulz orthogonalisation of each matrix of g [..., m, n] (bf16 or
    fp32, any strides): X = g / (|g|_F + eps), then `steps` times
    X <- a X + (b A + c A A) X with A = X X' (on the smaller side).  Returns
    bf16 X, contiguous, shaped like g (or `out`, which may be a contiguous bf16 g
    itself but not overlap it otherwise).

    coefficients: a triple (a, b, c) for all steps, or one for each.  They have
    to keep |X| within a few units (as the default and all schedules that
    converge do): X is held in 22 bits, its products have fp16 operands and fp32
    accumulators, and the result is within about 1e-3 of its definition before it
    is rounded to bf16.  |g|_F^2 is summed in 32 bits: |g|_F up to 1e19."""
    E, m, n, desc = _matrices(g, "g")
    dev = g.device
    if out is None:
        out = torch.empty_like(g, dtype=torch.bfloat16, memory_format=torch.contiguous_format)
    else:
        _check_out(out, "out", torch.bfloat16, dev, shape=g.shape)
        _check_replaces(out, "out", g, (g,))
    co = _schedule(steps, coefficients)
    with _on_device(dev):
        ws, ws_bytes, workspace = _workspace(workspace, orthogonalize_workspace_bytes(E, m, n), g)
        _lib.call("frag_orthogonalize", C.byref(desc), _ptr(out), E, m, n, steps, co, float(eps), ws, ws_bytes,
                  _stream(dev))
    return out


def muon_update(param: torch.Tensor, grad: torch.Tensor, momentum_buffer: torch.Tensor, *, lr: float,
                momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0, scale: float = 1.0,
                steps: int = 5, coefficients=NEWTON_SCHULZ, eps: float = 1e-7,
                param_out: torch.Tensor | None = None, momentum_out: torch.Tensor | None = None,
                workspace: torch.Tensor | None = None):
    """One weight update along the orthogonalised momentum of [..., m, n]
    matrices.  Returns (param', momentum'):

    momentum'  momentum * momentum_buffer + (1 - momentum) * grad
    u          momentum * momentum' + (1 - momentum) * grad (nesterov), or momentum'
    param'     (1 - lr * weight_decay) * param - lr * scale * orthogonalize(u)

    param, grad and momentum_buffer are bf16 or fp32, each its own; outputs are
    new contiguous tensors of param's and momentum_buffer's types, or the given
    param_out / momentum_out, which may be param and momentum_buffer themselves
    (an update in place).  steps, coefficients, eps as in orthogonalize.

    The step's own error, before param' is rounded: about 5e-4 of it (fp16
    operands), and 2e-6 where param is fp32, a matrix's one side is at most 128
    and the other at most 4096 (two fp16 numbers for each operand)."""
    E, m, n, dp = _matrices(param, "param")
    dev = param.device
    dg = _matrices(grad, "grad", dev, param.shape)[3]
    dm = _matrices(momentum_buffer, "momentum_buffer", dev, param.shape)[3]
    for v, name in ((lr, "lr"), (weight_decay, "weight_decay"), (scale, "scale"), (eps, "eps")):
        if not math.isfinite(v):
            raise ValueError(f"{name} must be finite")
    if not 0 <= momentum <= 1:
        raise ValueError("momentum must be in [0, 1]")
    outs = []
    for name, given, like in (("param_out", param_out, param), ("momentum_out", momentum_out, momentum_buffer)):
        if given is None:
            given = torch.empty_like(like, memory_format=torch.contiguous_format)
        else:
            _check_out(given, name, like.dtype, dev, shape=like.shape)
            _check_replaces(given, name, like, (param, grad, momentum_buffer))
        outs.append(given)
    if _overlaps(*outs):
        raise ValueError("param_out and momentum_out overlap")
    co = _schedule(steps, coefficients)
    with _on_device(dev):
        ws, ws_bytes, workspace = _workspace(workspace, orthogonalize_workspace_bytes(E, m, n), param)
        _lib.call("frag_muon_update", C.byref(dp), C.byref(dg), C.byref(dm), _ptr(outs[0]), _ptr(outs[1]), E, m, n,
                  float(lr), float(momentum), int(bool(nesterov)), float(weight_decay), float(scale), steps, co,
                  float(eps), ws, ws_bytes, _stream(dev))
    return outs[0], outs[1]


# ------------------------------------------------------------------ layer norm

# The ordinary call of these operators goes through the compiled binding: it
# checks, makes the outputs and launches in a third of the time.  What it does not
# take (None: strided rows, another device, anything to be refused) goes on in
# Python, to the same kernels.

def _taken(name: str, status) -> bool:
    """Whether the binding made the call; raises where the call failed."""
    if status is None:
        return False
    _lib.check(name, status)
    return True


def _norm_input(x: torch.Tensor, name: str):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if x.dtype not in _DT:
        raise TypeError(f"{name} must be bfloat16 or float32, got {x.dtype}")
    if not x.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if x.dim() < 1:
        raise ValueError(f"{name} must have at least one dimension")
    return x.shape[-1], x.dtype, x.device


def _norm_vectors(N: int, dev: torch.device, **vectors):
    """The vectors as contiguous [N] tensors or None, and the code of their one type."""
    out, dtype = [], None
    for name, v in vectors.items():
        if v is not None:
            if not isinstance(v, torch.Tensor) or v.dtype not in _DT or (dtype is not None and v.dtype != dtype):
                raise TypeError(f"{name} must be bfloat16 or float32, weight and bias of one type")
            dtype = v.dtype
            _need(v, name, dtype, dev)
            if v.numel() != N:
                raise ValueError(f"{name}: {v.numel()} elements, rows have {N}")
            v = v.contiguous()
        out.append(v)
    return (*out, _DT[dtype or torch.float32])


def _row_count(x: torch.Tensor, N: int) -> int:
    M = math.prod(x.shape[:-1])
    if N == 0 and M:
        raise ValueError("rows must hold at least one value")
    return M


def layernorm_fwd(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                  eps: float = 1e-5, *, residual: torch.Tensor | None = None, write_h: bool = True,
                  save_stats: bool = True):
    """(Residual add +) layer norm over the last dimension, in one pass.
    Returns (y, h, mean, rstd).

    y      (h - mean) * rstd * weight + bias, rounded once to x's type
    h      residual + x in x's type: the new residual stream, which the
           backward takes as its x; None without a residual or with write_h=False
    mean   fp32 x.shape[:-1], and
    rstd   1 / sqrt(mean((h - mean)^2) + eps), the same; None with save_stats=False

    x and residual: bf16 or fp32, rows of contiguous values, any row stride.
    weight, bias: bf16 or fp32 (both the same), or None for 1 and 0.

    Rows of up to 16384 values (14336 in fp32 with a residual) are read once, where those
    of x, residual and outputs (which begin at a 16-byte boundary) lie alike between such
    boundaries; any others two or three times, which takes up to four times as long.
    The mean is one fp32 number: y is off by up to |mean| 2^-24 rstd weight beside its
    own roundings."""
    out = _lib.binding().layernorm_fwd(x, weight, bias, eps, residual, write_h, save_stats)
    if out.__class__ is tuple:
        return out
    _taken("frag_layernorm_fwd", out)
    N, dtype, dev = _norm_input(x, "x")
    M = _row_count(x, N)
    x2, xs = _strided_rows(x, "x", N, dev, None, dtype)
    r2, rs = (None, 0) if residual is None else _strided_rows(residual, "residual", N, dev, x.shape, dtype)
    w, b, wdt = _norm_vectors(N, dev, weight=weight, bias=bias)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    h = mean = rstd = None
    if residual is not None and write_h:
        h = torch.empty_like(x, memory_format=torch.contiguous_format)
    if save_stats:
        mean, rstd = _new(x, x.shape[:-1], torch.float32), _new(x, x.shape[:-1], torch.float32)
    with _on_device(dev):
        _lib.call("frag_layernorm_fwd", _ptr(x2), xs, _ptr(r2), rs, _ptr(w), _ptr(b), _ptr(y), _ptr(h), _ptr(mean),
                  _ptr(rstd), M, N, float(eps), _DT[dtype], wdt, _stream(dev))
    return y, h, mean, rstd


def layernorm_bwd(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                  weight: torch.Tensor | None = None, *, dres: torch.Tensor | None = None, compute_dw: bool = True,
                  compute_db: bool = True, workspace: torch.Tensor | None = None):
    """The gradient of layernorm_fwd.  Returns (dx, dw, db).

    x      the normalised input (h of layernorm_fwd), mean and rstd its saved fp32
    dres   the residual stream's own gradient, added to dx
    dx     dres + the gradient of the norm, rounded once to x's type
    dw     fp32 [N], sum over the rows of dy * (x - mean) * rstd in a fixed order;
           None with compute_dw=False or without a weight
    db     fp32 [N], sum over the rows of dy in a fixed order; None with compute_db=False

    dy, x and dres: of one type, rows of contiguous values, any row stride; what
    layernorm_fwd says of rows that are read once holds here, with dres for residual."""
    if workspace is None:
        out = _lib.binding().layernorm_bwd(dy, x, mean, rstd, weight, dres, compute_dw, compute_db)
        if out.__class__ is tuple:
            return out
        _taken("frag_layernorm_bwd", out)
    N, dtype, dev = _norm_input(x, "x")
    M = _row_count(x, N)
    x2, xs = _strided_rows(x, "x", N, dev, None, dtype)
    y2, ys = _strided_rows(dy, "dy", N, dev, x.shape, dtype)
    r2, rs = (None, 0) if dres is None else _strided_rows(dres, "dres", N, dev, x.shape, dtype)
    for name, t in (("mean", mean), ("rstd", rstd)):
        _need(t, name, torch.float32, dev)
        if t.numel() != M or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous with {M} elements")
    w, wdt = _norm_vectors(N, dev, weight=weight)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    dw = x.new_empty(N, dtype=torch.float32) if compute_dw and weight is not None else None
    db = x.new_empty(N, dtype=torch.float32) if compute_db else None
    with _on_device(dev):
        need = int(_lib.load().frag_layernorm_bwd_workspace_bytes(M, N)) if dw is not None or db is not None else 0
        ws, ws_bytes, workspace = _workspace(workspace, need, x)
        _lib.call("frag_layernorm_bwd", _ptr(y2), ys, _ptr(x2), xs, _ptr(mean), _ptr(rstd), _ptr(w), _ptr(r2), rs,
                  _ptr(dx), _ptr(dw), _ptr(db), M, N, _DT[dtype], wdt, ws, ws_bytes, _stream(dev))
    return dx, dw, db


# -------------------------------------------------- many tensors in one launch

# A step's lists have hundreds of tensors: what is asked of each goes through
# map, 0.05 us a tensor and question where a loop of checks would take 1.
_dtype_of = operator.attrgetter("dtype")
_shape_of = operator.attrgetter("shape")


def _pointers(tensors) -> array:
    return array("Q", map(torch.Tensor.data_ptr, tensors))


def _address(a: array) -> int:
    return a.buffer_info()[0]


def _dense_list(tensors, name: str) -> torch.device:
    """Checks a list of contiguous bf16 or fp32 tensors on one CUDA device."""
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be tensors, got {type(t).__name__}")
    dtypes = set(map(_dtype_of, tensors))
    if not dtypes <= _DT.keys():
        raise TypeError(f"{name} must be bfloat16 or float32, got {sorted(map(str, dtypes - _DT.keys()))}")
    if not all(map(torch.Tensor.is_contiguous, tensors)):
        raise ValueError(f"{name} must be contiguous")
    devices = set(map(torch.Tensor.get_device, tensors))
    if len(devices) != 1:
        raise ValueError(f"{name} must be on one device")
    if devices == {-1}:
        raise ValueError(f"{name} must be CUDA tensors")
    return tensors[0].device


def _dtype_codes(tensors) -> array:
    dtypes = list(map(_dtype_of, tensors))
    first = dtypes[0] if dtypes else None
    if dtypes.count(first) == len(dtypes):
        return array("i", [_DT[first]] * len(dtypes)) if dtypes else array("i")
    return array("i", [_DT[d] for d in dtypes])


def grad_norm(grads, *, max_norm: float | None = None, workspace: torch.Tensor | None = None):
    """The 2-norm of a list of gradients together, and the factor that clips it,
    without a look from the host.  Returns (norm, scale), fp32 tensors of no
    dimension:

    norm   sqrt(sum of all squares), in an order that sizes and alignment alone decide
    scale  max_norm / max(norm, max_norm), which adamw_update takes as its
           grad_scale; NaN where norm is not finite (the update then changes
           nothing); None without max_norm

    grads: contiguous bf16 and fp32 tensors on one device, |g| up to 1e18 (and from 1e-18
    on: squares of smaller ones lose digits, and below 1e-22 count nothing); None entries
    are left out."""
    grads = list(grads)
    if workspace is None:
        out = _lib.binding().grad_norm(grads, max_norm)
        if out.__class__ is tuple:
            return out
        _taken("frag_grad_norm", out)
    grads = [g for g in grads if g is not None]
    if not grads:
        raise ValueError("grad_norm needs at least one tensor")
    if max_norm is not None and not (max_norm > 0 and math.isfinite(max_norm)):
        raise ValueError("max_norm must be positive and finite")
    dev = _dense_list(grads, "grads")
    ptrs, numel, codes = _pointers(grads), array("q", map(torch.Tensor.numel, grads)), _dtype_codes(grads)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    scale = None if max_norm is None else torch.empty((), dtype=torch.float32, device=dev)
    with _on_device(dev):
        need = int(_lib.load().frag_grad_norm_workspace_bytes(len(grads)))
        ws, ws_bytes, workspace = _workspace(workspace, need, norm)
        _lib.call("frag_grad_norm", _address(ptrs), _address(numel), _address(codes), len(grads),
                  1.0 if max_norm is None else float(max_norm), _ptr(norm), _ptr(scale), ws, ws_bytes, _stream(dev))
    return norm, scale


_F32_END = 2.0 ** 128 - 2.0 ** 103  # the least that 32 bits round to infinity


def _finite(v: float) -> bool:
    """Whether a number is finite in 32 bits."""
    return -_F32_END < v < _F32_END


def _each(v, n: int, name: str) -> list[float]:
    values = [float(v)] * n if isinstance(v, (int, float)) else [float(x) for x in v]
    if len(values) != n:
        raise ValueError(f"{name}: {len(values)} values for {n} tensors")
    if not all(map(_finite, values)):
        raise ValueError(f"{name} must be finite, in 32 bits")
    return values


def _disjoint(tensors, name: str) -> None:
    """Refuses contiguous tensors that share memory."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors if t.numel())
    for (_, end), (start, _) in zip(spans, spans[1:]):
        if start < end:
            raise ValueError(f"{name} share memory")


class AdamWStates:
    """The moments of a list of parameters for adamw_update, and what is fixed
    about each parameter.

    params        contiguous bf16 or fp32 CUDA tensors of one device, updated in place
    dtype         torch.float32, or torch.float8_e4m3fn: 8 bits and a scale for
                  each 128 values of a tensor, for betas up to (0.95, 0.98)
    weight_decay  one for all, or one for each (0 for norms and biases)
    lr_scale      a factor on lr, one for all or one for each
    copies        bf16 tensors (or None) shaped like the parameters, which receive
                  the rounded parameter in the same pass: the model's weights where
                  the parameters are their fp32 masters

    States are flat tensors, zero at first; parameter i's begin at offsets[i] (a
    multiple of 128), and the values behind its end are zero:
      exp_avg, exp_avg_sq               fp32: first and second moment
      exp_avg, exp_avg_scale,           8 bits: the first moment and the root of the
      exp_avg_sq, exp_avg_sq_scale      second, each value * scale[its index // 128]
    A tensor's place in memory is looked up in every call, so a parameter whose data
    was replaced (by one of the same shape and type) is found again."""

    GROUP = 128

    def __init__(self, params, *, dtype: torch.dtype = torch.float32, weight_decay=0.0, lr_scale=1.0, copies=None):
        self.params = tuple(params)
        n = len(self.params)
        if not n:
            raise ValueError("AdamWStates needs at least one parameter")
        if dtype not in (torch.float32, torch.float8_e4m3fn):
            raise TypeError("dtype must be float32 or float8_e4m3fn")
        decay, lr_scale = _each(weight_decay, n, "weight_decay"), _each(lr_scale, n, "lr_scale")
        self._most_scale = max(1.0, *map(abs, lr_scale))
        self.device = _dense_list(self.params, "params")
        self.copies = (None,) * n if copies is None else tuple(copies)
        if len(self.copies) != n:
            raise ValueError(f"copies: {len(self.copies)} for {n} parameters")
        for p, c in zip(self.params, self.copies):
            if c is not None:
                _check_out(c, "a copy", torch.bfloat16, self.device, shape=p.shape)
        self.dtype = dtype
        self._shapes = list(map(_shape_of, self.params))
        self._written = [*self.params, *(c for c in self.copies if c is not None)]
        self._kinds = list(map(_dtype_of, self._written))
        self._numel = list(map(torch.Tensor.numel, self._written))
        _disjoint(self._written, "parameters and copies")
        self.offsets, total = [], 0
        for numel in self._numel[:n]:
            self.offsets.append(total)
            total += -(-numel // self.GROUP) * self.GROUP
        self._total = total
        self.exp_avg = torch.zeros(total, dtype=dtype, device=self.device)
        self.exp_avg_sq = torch.zeros(total, dtype=dtype, device=self.device)
        self.exp_avg_scale = self.exp_avg_sq_scale = None
        if dtype != torch.float32:
            self.exp_avg_scale = torch.ones(total // self.GROUP, dtype=torch.float32, device=self.device)
            self.exp_avg_sq_scale = torch.ones_like(self.exp_avg_scale)
        self._table = (_lib.AdamWTensor * n)()
        for i, e in enumerate(self._table):
            e.numel, e.state_offset = self._numel[i], self.offsets[i]
            e.lr_scale, e.weight_decay, e.param_dtype = lr_scale[i], decay[i], _DT[self._kinds[i]]
        self._codes, self._counts = _dtype_codes(self._written), array("q", self._numel)
        self._places = None
        self._place()

    def _place(self) -> None:
        """The table's addresses, looked up again; checked where any has changed."""
        written = self._written
        if (list(map(_dtype_of, written)) != self._kinds or list(map(torch.Tensor.numel, written)) != self._numel
                or not all(map(torch.Tensor.is_contiguous, written))):
            raise ValueError("a parameter or copy has another type or shape than the states were made for")
        places = _pointers(written)
        if places == self._places:
            return
        if _dense_list(written, "params") != self.device:
            raise ValueError(f"parameters are no longer on {self.device}")
        if list(map(_shape_of, self.params)) != self._shapes:
            raise ValueError("a parameter has another shape than the states were made for")
        _disjoint(written, "parameters and copies")
        at = len(self.params)
        for i, e in enumerate(self._table):
            e.param, e.copy = places[i], None
            if self.copies[i] is not None:
                e.copy = places[at]
                at += 1
        self._places = places
        # what the binding compares the tensors with: addresses of the three arrays, and the table's
        self._known = (written, _address(places), _address(self._codes), _address(self._counts)), C.addressof(self._table)

    def _held(self):
        """The states' addresses; refused where one is not what it was made as."""
        total, out = self._total, []
        for k, dtype, numel in (("exp_avg", self.dtype, total), ("exp_avg_sq", self.dtype, total),
                                ("exp_avg_scale", torch.float32, total // self.GROUP),
                                ("exp_avg_sq_scale", torch.float32, total // self.GROUP)):
            t = getattr(self, k)
            if k.endswith("scale") and self.dtype == torch.float32:
                out.append(None)
            else:
                out.append(_check_out(t, k, dtype, self.device, numel=numel).data_ptr())
        return out

    def moments(self, i: int):
        """Parameter i's first and second moment, new fp32 tensors of its shape."""
        a, n, shape = self.offsets[i], self._numel[i], self._shapes[i]
        held = slice(a, a + -(-n // self.GROUP) * self.GROUP)
        m, v = self.exp_avg[held].float(), self.exp_avg_sq[held].float()
        if self.dtype != torch.float32:
            at = slice(held.start // self.GROUP, held.stop // self.GROUP)
            m = (m.view(-1, self.GROUP) * self.exp_avg_scale[at, None]).view(-1)
            v = (v.view(-1, self.GROUP) * self.exp_avg_sq_scale[at, None]).view(-1).square()
        return m[:n].clone().view(shape), v[:n].clone().view(shape)

    _NAMES = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")

    def state_dict(self) -> dict:
        """The states themselves (not copies), by name, and the sizes they are for."""
        d = {k: getattr(self, k) for k in self._NAMES if getattr(self, k) is not None}
        return {"numel": self._numel[:len(self.params)], **d}

    def load_state_dict(self, d: dict) -> None:
        if list(d["numel"]) != self._numel[:len(self.params)]:
            raise ValueError("the states are of parameters of other sizes")
        held = [k for k in self._NAMES if getattr(self, k) is not None]
        if {k for k in self._NAMES if d.get(k) is not None} != set(held) or any(
                d[k].dtype != getattr(self, k).dtype or d[k].shape != getattr(self, k).shape for k in held):
            raise ValueError("the states are of another type or shape")
        for k in held:
            getattr(self, k).copy_(d[k])


def _device_word(t: torch.Tensor, name: str, dtype: torch.dtype, dev: torch.device) -> int:
    _need(t, name, dtype, dev)
    if t.numel() != 1:
        raise ValueError(f"{name} must have one element")
    return t.data_ptr()


def adamw_update(states: AdamWStates, grads, *, lr, step, betas=(0.9, 0.95), eps: float = 1e-8,
                 grad_scale: torch.Tensor | None = None) -> None:
    """One AdamW step over all parameters of `states` in one launch, in place
    (parameters, their bf16 copies, and states):

      g  grad_scale * grad
      m  beta1 * m + (1 - beta1) * g,   v  beta2 * v + (1 - beta2) * g^2
      p  (1 - l * weight_decay) * p - l * m / (1 - beta1^step) / (sqrt(v / (1 - beta2^step)) + eps)
         with l = lr * lr_scale

    grads       a tensor for each parameter, of its shape, contiguous, bf16 or fp32;
                None leaves that parameter and its states as they are
    lr          a number, or a one-element fp32 CUDA tensor
    step        counts from 1: an int, or a one-element int64 CUDA tensor, which a
                captured call reads anew in every replay (an int and a float lr
                are what they were at capture)
    grad_scale  one-element fp32 CUDA tensor (grad_norm's scale), or None

    Where grad_scale or a device lr is not finite (times a tensor's lr_scale, in 32 bits), or
    a device step below 1, nothing is changed.  Parameters are rounded to nearest: bf16 ones do not move by less than
    2^-9 of their value, for which there are fp32 parameters with bf16 copies.  With
    states in 8 bits a gradient that is not finite makes its whole group of 128 NaN.

    States in 8 bits are rounded to nearest, too: one moves by itself only where a step
    moves it by over half of E4M3's step (3 to 6 percent), and else with its group, whose
    scale is fp32.  What decays more slowly stays behind a value that holds the scale.
    With a group's gradients fallen tenfold but for one value's, the others' roots of the
    second moment are, 20 / (1 - beta2) steps later, 1.0 times what they should be at
    beta2 = 0.95, 1.04 at 0.98, 5.9 at 0.99 and 7.7 at 0.999, and their steps as many times
    too small.  Roots of values whose gradients end stay on at any beta2, which changes
    nothing until they come again; first moments of such values go at beta1 = 0.9, and
    beside a value that does not change up to a twentieth of them stays at 0.95, half at
    0.97.  So above betas of (0.95, 0.98) there is a warning: those are for states in 32 bits.
    Gradients must not share memory with parameters, copies or states."""
    if not isinstance(states, AdamWStates):
        raise TypeError("states must be an AdamWStates")
    dev = states.device
    n = len(states.params)
    grads = list(grads)
    if len(grads) != n:
        raise ValueError(f"{len(grads)} gradients for {n} parameters")
    b1, b2 = betas
    if not (0 <= b1 < 1 and 0 <= b2 < 1):
        raise ValueError("betas must be in [0, 1)")
    if (b1 > 0.95 or b2 > 0.98) and states.dtype != torch.float32:
        warnings.warn(f"states in 8 bits stay behind with betas of ({b1}, {b2}): above (0.95, 0.98) take float32",
                      RuntimeWarning, stacklevel=2)
    if not (eps >= 2.0 ** -126 and math.isfinite(eps)):
        raise ValueError("eps must be finite and at least 2^-126, the least normal number of 32 bits")
    lr_t = step_t = None
    if isinstance(lr, torch.Tensor):
        lr_t, lr = lr, 0.0
    elif not _finite(lr * states._most_scale):
        raise ValueError("lr must be finite, in 32 bits and times every lr_scale")
    if isinstance(step, torch.Tensor):
        step_t, step = step, 0
    elif not isinstance(step, int) or step < 1:
        raise ValueError("step must be an int from 1 on")
    known, table = states._known
    if _taken("frag_adamw_update", _lib.binding().adamw(
            *known, grads, table, states.exp_avg, states.exp_avg_sq, states.exp_avg_scale, states.exp_avg_sq_scale,
            states._total, lr, lr_t, b1, b2, eps, step, step_t, grad_scale)):
        return
    lr_ptr = None if lr_t is None else _device_word(lr_t, "lr", torch.float32, dev)
    step_ptr = None if step_t is None else _device_word(step_t, "step", torch.int64, dev)
    scale_ptr = None if grad_scale is None else _device_word(grad_scale, "grad_scale", torch.float32, dev)
    shapes = states._shapes
    if any(g is None for g in grads):
        given = [g for g in grads if g is not None]
        shapes = [s for s, g in zip(shapes, grads) if g is not None]
        if not given:
            return
    else:
        given = grads
    if _dense_list(given, "grads") != dev:
        raise ValueError(f"grads must be on {dev}")
    if list(map(_shape_of, given)) != shapes:
        raise ValueError("every gradient must have its parameter's shape")
    states._place()
    if given is grads:
        ptrs, codes = _pointers(grads), _dtype_codes(grads)
    else:
        ptrs = array("Q", [0 if g is None else g.data_ptr() for g in grads])
        codes = array("i", [0 if g is None else _DT[g.dtype] for g in grads])
    with _on_device(dev):
        _lib.call("frag_adamw_update", states._table, _address(ptrs), _address(codes), n, *states._held(), float(lr),
                  lr_ptr, float(b1), float(b2), float(eps), step, step_ptr, scale_ptr, _stream(dev))
