"""Operator-level Python entry points: torch tensors in, C-ABI calls out.

Torch is used for device memory and the current stream only; all arithmetic
happens inside libchitu_b200.so.  Every function raises if the tensors are not
on a CUDA device - there is no CPU path.
"""

from __future__ import annotations

import ctypes
import functools
import math
import os
import threading
from typing import Optional, Sequence, Tuple

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, torch.float32: _lib.DTYPE_FP32}

_STATUS_NAMES = {
    1: "TMA producer waited too long for a free K/V stage",
    2: "MMA issuer waited too long for operands",
    3: "softmax warps waited too long for scores",
    4: "epilogue waited too long for the last MMA",
    5: "a bounded flag wait ran out",
}

_status_words = {}

_workspaces = {}
_retired_workspaces = []
_cut_scratches = {}
_scratch_lock = threading.Lock()

# kernels of this library launched so far by this process (the bench reports the count of a timed region)
launch_count = 0


def _launched(n: int = 1) -> None:
    global launch_count
    launch_count += n


# the devices that tensors carry (a look-up costs a third of asking the object for its type and index)
_CUDA_INDEX = {torch.device("cuda", i): i for i in range(64)}


def _device_key(device) -> int:
    """Index of a device given in any of the forms torch takes: an object, a name, an index, None for the current one."""
    index = _CUDA_INDEX.get(device)
    if index is not None:
        return index
    if not isinstance(device, torch.device):
        device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise ValueError(f"Expected a cuda device, but got: {device}")
    return torch.cuda.current_device() if device.index is None else device.index


def _stream_ptr(device) -> int:
    # the handle alone: building a torch Stream object costs ten times as much and every call needs it
    index = _CUDA_INDEX.get(device)
    return torch._C._cuda_getCurrentRawStream(_device_key(device) if index is None else index)


class _NoGuard:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_NO_GUARD = _NoGuard()


def _on(device):
    """``torch.cuda.device(device)`` where that changes anything (entering and leaving it costs some microseconds)."""
    index = _CUDA_INDEX.get(device)
    if index is not None and torch._C._cuda_getDevice() == index:
        return _NO_GUARD
    return torch.cuda.device(device)


def _require_cuda(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError("chitudiffusion_b200 runs on CUDA tensors only (there is no CPU path)")


def status_word(device: torch.device) -> torch.Tensor:
    """Per-device int32 status word that kernels with bounded waits report into.

    It lives in pinned host memory, which kernels address directly: a wait that ran out is stored there and the host
    looks at it without a copy, an event or a synchronisation in between.
    """
    key = _device_key(device)
    entry = _status_words.get(key)
    if entry is None:
        word = torch.zeros(1, dtype=torch.int32, pin_memory=True)
        entry = _status_words.setdefault(key, (word, ctypes.c_int32.from_address(word.data_ptr())))
    return entry[0]


def _take_status(key: int) -> None:
    """Raise (and clear the word) if it is set.  A call that gave up may have left counters in its scratch that no later
    call completes, so the device's buffers are not used again."""
    entry = _status_words.get(key)
    if entry is not None and entry[1].value != 0:
        code = entry[1].value
        entry[1].value = 0
        with _scratch_lock:
            for used in [k for k in _workspaces if k[0] == key]:
                _retired_workspaces.append(_workspaces.pop(used))
            for used in [k for k in _cut_scratches if k[0] == key]:
                del _cut_scratches[used]
        raise _lib.ChituB200Error(f"device status {code}: {_STATUS_NAMES.get(code, 'unknown')}")


def check_status(device: Optional[torch.device] = None) -> None:
    """Synchronise and raise if any kernel on `device` reported a timed-out wait.

    The scratch buffers that this module keeps for the device are then replaced.  A buffer that the caller passed as
    ``workspace=`` is the caller's to clear: zero its first ``SPLIT_HEADER_BYTES`` before it is used again."""
    key = torch.cuda.current_device() if device is None else _device_key(device)
    torch.cuda.synchronize(key)
    _take_status(key)


def poll_status(device: Optional[torch.device] = None) -> None:
    """Deferred, non-blocking form of :func:`check_status` for the product path.

    Looks at the status word as it is: a device wait that timed out surfaces as an exception at the first call after
    its kernel has reported it, instead of as silently wrong output, and no call ever synchronises or enqueues
    anything.  ``CHITU_B200_CHECK=1`` makes every poll a full synchronising check.  Does nothing while the stream is
    being captured.
    """
    key = torch.cuda.current_device() if device is None else _device_key(device)
    entry = _status_words.get(key)
    checking = os.environ.get("CHITU_B200_CHECK", "0") == "1"
    if (checking or (entry is not None and entry[1].value != 0)) and not torch.cuda.is_current_stream_capturing():
        if checking:
            torch.cuda.synchronize(key)
        _take_status(key)


def set_flag_wait_cycles(cycles: int) -> int:
    """Clock budget of the cross-GPU flag waits; returns the previous one (see ``chitu_b200_set_flag_wait_cycles``)."""
    return int(_lib.load().chitu_b200_set_flag_wait_cycles(int(cycles)))


NUM_SMS = 148

SPLIT_HEADER_BYTES = 65536  # counters at the head of every scratch buffer (CHITU_SPLITKV_HEADER_BYTES)
# what the largest cut needs on NUM_SMS SMs: a bundle per SM, each with two fragments of two 128-row tiles
CUT_SCRATCH_BYTES = SPLIT_HEADER_BYTES + NUM_SMS * 4 * 128 * (128 + 1) * 4
CUT_SCRATCH_STREAMS = 8


def auto_key_splits(B: int, Sq: int, Sk: int, H: int) -> int:
    """How many key ranges to run as separate CTAs.  A CTA serves 256 query rows of one head; the grid runs in
    waves of one CTA per SM, so the cost of a call is (waves) x (key tiles per CTA, plus about 5 tile steps for
    a CTA's prologue and for parking its partial rows: 216 CTAs x 36 tiles measured 138 us, 432 CTAs x 18 tiles
    143 us) plus about one tile step per range for the merge.  The split that minimises it is taken when it
    saves at least 8 %: it fills small grids (54 CTAs -> 2 ranges).  The model is that of ``attn_fwd_kernel``: it knows neither
    the persistent kernel of plain calls above one wave nor the cut of its last wave, and still splits some grids
    of 149 to about 220 blocks that the cut would serve better (150 x 60 tiles: two ranges 176 us, cut 135).
    ``CHITU_B200_KEY_SPLITS`` overrides."""
    forced = os.environ.get("CHITU_B200_KEY_SPLITS")
    tiles = -(-Sk // 128)
    if forced:
        return max(1, min(int(forced), tiles, 64))
    return _wave_model_splits(-(-Sq // 256) * H * B, tiles)


@functools.lru_cache(maxsize=1024)
def _wave_model_splits(ctas: int, tiles: int) -> int:
    def cost(n):
        per = -(-tiles // n)
        n_eff = -(-tiles // per)
        waves = -(-ctas * n_eff // NUM_SMS)
        return waves * per if n_eff == 1 else waves * (per + 5.0) + 1.0 * n_eff

    best, best_cost = 1, cost(1)
    for n in range(2, min(tiles, 16) + 1):
        if ctas * n > 512:  # the parked rows (128 KiB per CTA) should stay in L2 until they are merged
            break
        c = cost(n)
        if c < best_cost * 0.92 and c < cost(best):
            best, best_cost = n, c
    return best


def splitkv_workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """Scratch for key-split partials, one buffer per (device, stream), grown on demand, zero-filled when
    created (the library keeps per-query-block counters in its first 64 KiB and leaves them zero after each call).

    A buffer that has been handed out may have been passed to a captured call as ``workspace=``, so a superseded
    buffer is never freed: it is parked for the life of the process and the larger replacement serves later
    calls.  Streams do not share a buffer (two streams of one GPU may run key-split calls at once).  Calls of this
    module that are captured do not use it (see :func:`_split_scratch`), and objects that own long-lived graphs (the
    peer exchanges) allocate their own scratch and pass it as ``workspace=``.
    """
    dev = torch.device(device)
    key = (dev.index if dev.index is not None else torch.cuda.current_device(),
           int(torch.cuda.current_stream(dev).cuda_stream))
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        if ws is not None:
            _retired_workspaces.append(ws)
        ws = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=dev)  # the counters at its head start at zero
        with _scratch_lock:
            _workspaces[key] = ws
    return ws


def _split_scratch(device: torch.device, nbytes: int) -> torch.Tensor:
    """Key-split scratch of one call on the current stream of ``device``.

    A call that is being captured gets its own, from the graph's memory and with its counters cleared by the graph
    itself: a replay runs on any stream, beside eager calls of this one, and memory that is first zeroed by a replay
    is not zero for an eager call before it.
    """
    with _on(device):
        if not torch.cuda.is_current_stream_capturing():
            return splitkv_workspace(device, nbytes)
        ws = torch.empty(max(nbytes, SPLIT_HEADER_BYTES), dtype=torch.uint8, device=device)
        ws[:SPLIT_HEADER_BYTES].zero_()
        return ws


def _cut_scratch(device: torch.device, nbytes: int) -> torch.Tensor:
    """Scratch for the cut query blocks of eager calls on the current stream of ``device``, and for attention over a cache.

    Never the buffer of :func:`splitkv_workspace`, whose address a caller's captured graph may hold.  A cut's need has a
    bound, so the buffer is made once at that size (39 MB; cache attention's bound is 0.4 MB above it).  The buffers made
    last are kept; an older one goes back to torch's allocator, which reuses it in its stream's order.  None is kept past a
    wait that ran out (see :func:`check_status`).
    """
    key = (_device_key(device), _stream_ptr(device))
    ws = _cut_scratches.get(key)
    if ws is None or ws.numel() < nbytes:
        with _on(device):
            ws = torch.empty(max(nbytes, CUT_SCRATCH_BYTES), dtype=torch.uint8, device=device)
            ws[:SPLIT_HEADER_BYTES].zero_()
        with _scratch_lock:
            _cut_scratches.pop(key, None)
            _cut_scratches[key] = ws
            while len(_cut_scratches) > CUT_SCRATCH_STREAMS:
                _cut_scratches.pop(next(iter(_cut_scratches)))
    return ws


def _holds(ws: torch.Tensor, nbytes: int, device: torch.device) -> bool:
    """Whether a caller's buffer will do as scratch of a call that can also run without (a call on one key range has
    always taken any ``workspace``, and left it alone)."""
    return (ws.device == device and ws.numel() * ws.element_size() >= nbytes and ws.data_ptr() % 16 == 0
            and ws.is_contiguous())


def splitkv_workspace_bytes(B: int, Sq: int, H: int, D: int, n_splits: int) -> int:
    """Bytes of scratch a key-split call of this shape needs (0 for one split)."""
    return int(_lib.load().chitu_b200_attn_splitkv_workspace_bytes(B, Sq, H, D, int(n_splits)))


@functools.lru_cache(maxsize=1024)
def _balanced_workspace_bytes(device_index: int, B: int, Sq: int, Sk: int, H: int) -> int:
    with torch.cuda.device(device_index):
        return int(_lib.load().chitu_b200_attn_balanced_workspace_bytes(B, Sq, Sk, H))


def attn_fwd(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    softmax_scale: Optional[float] = None,
    return_lse: bool = False,
    out: Optional[torch.Tensor] = None,
    n_splits: Optional[int] = None,
    workspace: Optional[torch.Tensor] = None,
    q_pre: Optional[dict] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``softmax(scale * q k^T) v`` for ``[B,S,H,128]`` bf16/fp16 tensors of any (16-byte aligned) strides.

    Returns ``(out [B,Sq,H,D] contiguous, lse [B,H,Sq] fp32 | None)``.  ``workspace`` is an optional
    caller-owned uint8 scratch for the key-split partials (see :func:`splitkv_workspace`) and for the cut query blocks of
    a call on one key range, which is not cut where the buffer will not do; its first 64 KiB
    hold counters that must be zero before the first use (``torch.zeros``) and are left zero by every call.  With ``q_pre``
    (keys ``norm_mode, rope_mode, weight, rstd, eps, rope_table, grid, axis_split, pos_offset, round_mid``)
    ``q`` is the raw projection and its pre-attention transform runs inside the kernel
    (``chitu_b200_attn_fwd_qpre``).
    """
    _require_cuda(q, k, v)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k, v must be [B, S, H, D]")
    B, Sq, H, D = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[2] != H or k.shape[3] != D:
        raise ValueError(f"shape mismatch: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise NotImplementedError("attention kernel takes bf16 or fp16 q/k/v of one dtype")
    Sk = k.shape[1]
    if Sq == 0 or Sk == 0:
        raise ValueError("empty sequence")

    def usable(t):
        return t.stride(3) == 1 and all(s % 8 == 0 for s in t.stride()[:3]) and t.data_ptr() % 16 == 0

    q, k, v = (t if usable(t) else t.contiguous() for t in (q, k, v))
    if out is None:
        out = torch.empty((B, Sq, H, D), dtype=q.dtype, device=q.device)
    elif out.shape != (B, Sq, H, D) or not out.is_contiguous() or out.dtype != q.dtype:
        raise ValueError("out must be a contiguous [B,Sq,H,D] tensor of q's dtype")
    lse = torch.empty((B, H, Sq), dtype=torch.float32, device=q.device) if return_lse else None
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(D)
    lib = _lib.load()
    automatic = n_splits is None
    if automatic:
        n_splits = auto_key_splits(B, Sq, Sk, H)
    if q_pre is not None:
        w, rstd, table = q_pre.get("weight"), q_pre.get("rstd"), q_pre.get("rope_table")
        _require_cuda(w, rstd, table)
        if w is not None:
            w = w.contiguous()
        grid = q_pre.get("grid", (0, 0, 0))
        split = q_pre.get("axis_split", (0, 0))
        desc = _lib.QPre(
            int(q_pre.get("norm_mode", 2)), int(q_pre.get("rope_mode", 0)), 1 if q_pre.get("round_mid", True) else 0,
            _DTYPES[w.dtype] if w is not None else _lib.DTYPE_FP32, w.data_ptr() if w is not None else None,
            rstd.data_ptr() if rstd is not None else None, float(q_pre.get("eps", 1e-6)),
            table.data_ptr() if table is not None else None, int(table.shape[0]) if table is not None else 0,
            int(grid[0]), int(grid[1]), int(grid[2]), int(split[0]), int(split[1]), int(q_pre.get("pos_offset", 0)))
        ws_ptr, ws_bytes = None, 0
        if n_splits > 1:
            need = int(lib.chitu_b200_attn_splitkv_workspace_bytes(B, Sq, H, D, n_splits))
            ws = workspace if workspace is not None else _split_scratch(q.device, need)
            ws_ptr, ws_bytes = ws.data_ptr(), ws.numel()
        with _on(q.device):
            rc = lib.chitu_b200_attn_fwd_qpre(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else None,
                B, Sq, Sk, H, D, _lib.i64_array(q.stride()), _lib.i64_array(k.stride()), _lib.i64_array(v.stride()),
                scale, _DTYPES[q.dtype], ctypes.byref(desc), int(n_splits), ws_ptr, ws_bytes,
                status_word(q.device).data_ptr(), _stream_ptr(q.device))
        _lib.check(rc, "attn_fwd_qpre")
        _launched(1)
        return out, lse
    with _on(q.device):
        if n_splits > 1:
            need = int(lib.chitu_b200_attn_splitkv_workspace_bytes(B, Sq, H, D, n_splits))
            ws = workspace if workspace is not None else _split_scratch(q.device, need)
            if ws.numel() * ws.element_size() < need or ws.device != q.device:
                raise ValueError(f"attn_fwd: workspace must hold {need} bytes on {q.device}")
            rc = lib.chitu_b200_attn_fwd_splitkv(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                lse.data_ptr() if lse is not None else None, B, Sq, Sk, H, D, _lib.i64_array(q.stride()),
                _lib.i64_array(k.stride()), _lib.i64_array(v.stride()), scale, _DTYPES[q.dtype], int(n_splits),
                ws.data_ptr(), ws.numel(), status_word(q.device).data_ptr(), _stream_ptr(q.device),
            )
        else:
            # the query blocks of a partly filled last wave are cut along the keys; a graph being captured
            # keeps them whole (their scratch belongs to eager calls of this stream, which may run beside a replay)
            ws_ptr, ws_bytes = None, 0
            if automatic and not torch.cuda.is_current_stream_capturing():
                need = _balanced_workspace_bytes(q.device.index, B, Sq, Sk, H)
                if need:
                    ws = _cut_scratch(q.device, need) if workspace is None else workspace
                    if _holds(ws, need, q.device):
                        ws_ptr, ws_bytes = ws.data_ptr(), ws.numel() * ws.element_size()
            rc = lib.chitu_b200_attn_fwd_balanced(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                lse.data_ptr() if lse is not None else None, B, Sq, Sk, H, D, _lib.i64_array(q.stride()),
                _lib.i64_array(k.stride()), _lib.i64_array(v.stride()), scale, _DTYPES[q.dtype], ws_ptr, ws_bytes,
                status_word(q.device).data_ptr(), _stream_ptr(q.device),
            )
    _lib.check(rc, "attn_fwd")
    _launched(1)
    return out, lse


def attn_fwd_q8(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    softmax_scale: Optional[float] = None,
    return_lse: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Quantised attention (INT8 QK^T, E4M3 PV); see ``chitu_b200_attn_fwd_q8``."""
    _require_cuda(q, k, v)
    B, Sq, H, D = q.shape
    Sk = k.shape[1]
    if k.shape != v.shape or k.shape[0] != B or k.shape[2] != H or k.shape[3] != D:
        raise ValueError(f"shape mismatch: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise NotImplementedError("attention kernel takes bf16 or fp16 q/k/v of one dtype")

    def usable(t):
        return t.stride(3) == 1 and all(s % 4 == 0 for s in t.stride()[:3]) and t.data_ptr() % 16 == 0

    q, k, v = (t if usable(t) else t.contiguous() for t in (q, k, v))
    out = torch.empty((B, Sq, H, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, H, Sq), dtype=torch.float32, device=q.device) if return_lse else None
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(D)
    lib = _lib.load()
    need = int(lib.chitu_b200_attn_q8_workspace_bytes(B, Sq, Sk, H))
    ws = torch.empty(need + 256, dtype=torch.uint8, device=q.device)
    base = (ws.data_ptr() + 255) // 256 * 256
    with _on(q.device):
        rc = lib.chitu_b200_attn_fwd_q8(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else None,
            B, Sq, Sk, H, D, _lib.i64_array(q.stride()), _lib.i64_array(k.stride()), _lib.i64_array(v.stride()),
            scale, _DTYPES[q.dtype], base, need, status_word(q.device).data_ptr(), _stream_ptr(q.device),
        )
    _lib.check(rc, "attn_fwd_q8")
    _launched(3)
    return out, lse


def lse_combine(
    acc_out: torch.Tensor,
    acc_lse: torch.Tensor,
    block_out: torch.Tensor,
    block_lse: torch.Tensor,
    first: bool,
    final_out: Optional[torch.Tensor] = None,
) -> None:
    """In-place fold of one partial result; see ``chitu_b200_lse_combine``.

    ``acc_out [B,S,H,D] fp32``, ``acc_lse [B,S,H]`` (or ``[B,S,H,1]``) fp32, ``block_out [B,S,H,D]``,
    ``block_lse [B,H,S] fp32``; all contiguous.
    """
    _require_cuda(acc_out, acc_lse, block_out, block_lse, final_out)
    B, S, H, D = block_out.shape
    if acc_out.shape != block_out.shape or acc_out.dtype != torch.float32 or not acc_out.is_contiguous():
        raise ValueError("acc_out must be contiguous fp32 [B,S,H,D]")
    if acc_lse.numel() != B * S * H or acc_lse.dtype != torch.float32 or not acc_lse.is_contiguous():
        raise ValueError("acc_lse must be contiguous fp32 [B,S,H] or [B,S,H,1]")
    if tuple(block_lse.shape) != (B, H, S) or block_lse.dtype != torch.float32:
        raise ValueError("block_lse must be fp32 [B,H,S]")
    block_out = block_out.contiguous()
    block_lse = block_lse.contiguous()
    if final_out is not None and (final_out.shape != block_out.shape or not final_out.is_contiguous()):
        raise ValueError("final_out must be contiguous [B,S,H,D]")
    lib = _lib.load()
    with _on(acc_out.device):
        rc = lib.chitu_b200_lse_combine(
            acc_out.data_ptr(), acc_lse.data_ptr(), block_out.data_ptr(), block_lse.data_ptr(), B, S, H, D,
            _DTYPES[block_out.dtype], 1 if first else 0,
            final_out.data_ptr() if final_out is not None else None,
            _DTYPES[final_out.dtype] if final_out is not None else 0, _stream_ptr(acc_out.device),
        )
    _lib.check(rc, "lse_combine")
    _launched()


def qk_norm_rope(
    x: torch.Tensor,
    num_heads: int,
    weight: Optional[torch.Tensor],
    eps: float,
    norm_mode: int,
    rope_mode: int,
    rope_table: Optional[torch.Tensor],
    grid: Sequence[int] = (0, 0, 0),
    axis_split: Sequence[int] = (0, 0),
    pos_offset: int = 0,
    out: Optional[torch.Tensor] = None,
    out_strides: Optional[Sequence[int]] = None,
    heads_per_group: Optional[int] = None,
    out_dtype: torch.dtype = torch.bfloat16,
    round_mid: bool = True,
    out_ptrs: Optional[Sequence[int]] = None,
) -> Optional[torch.Tensor]:
    """RMSNorm + rotary + 16-bit cast of a projection output ``[B,S,H*D]``; see ``chitu_b200_qk_norm_rope``.

    Without ``out`` a contiguous ``[B,S,H,D]`` tensor is returned.  With ``out`` and ``out_strides``
    ``(b, s, head_group, head_in_group)`` the result is scattered into a caller-owned buffer.
    """
    _require_cuda(x, weight, rope_table, out)
    if x.dim() != 3:
        raise ValueError("x must be [B, S, C]")
    B, S, C = x.shape
    if C % num_heads:
        raise ValueError("channels not divisible by num_heads")
    D = C // num_heads
    if x.stride(2) != 1 or (B > 1 and x.stride(0) != S * x.stride(1)):
        x = x.contiguous()
    if weight is not None:
        weight = weight.contiguous()
        if weight.dtype not in _DTYPES:
            raise ValueError("weight dtype must be bf16, fp16 or fp32")
    if rope_mode != 0:
        if rope_table is None or rope_table.dtype != torch.float32 or not rope_table.is_contiguous():
            raise ValueError("rope_table must be a contiguous fp32 [rows, D/2, 2] tensor")
        if rope_table.shape[-2:] != (D // 2, 2):
            raise ValueError(f"rope_table must be [rows, {D // 2}, 2]")
    if out_ptrs is not None:
        if out is not None or out_strides is None or heads_per_group is None:
            raise ValueError("out_ptrs needs out_strides and heads_per_group, and excludes out")
    elif out is None:
        out = torch.empty((B, S, num_heads, D), dtype=out_dtype, device=x.device)
        out_strides = (S * C, C, 0, D)
        heads_per_group = num_heads
    elif out_strides is None or heads_per_group is None:
        raise ValueError("out needs out_strides and heads_per_group")
    lib = _lib.load()
    split = (ctypes.c_int * 2)(int(axis_split[0]), int(axis_split[1]))
    common = (
        x.data_ptr(), _DTYPES[x.dtype], x.stride(1), weight.data_ptr() if weight is not None else None,
        _DTYPES[weight.dtype] if weight is not None else _lib.DTYPE_FP32, float(eps), int(norm_mode),
        int(rope_mode), rope_table.data_ptr() if rope_table is not None else None,
        int(rope_table.shape[0]) if rope_table is not None else 0, int(grid[0]), int(grid[1]), int(grid[2]),
        split, int(pos_offset),
    )
    tail = (_lib.i64_array(out_strides), int(heads_per_group), B, S, num_heads, D, 1 if round_mid else 0,
            _stream_ptr(x.device))
    with _on(x.device):
        if out_ptrs is not None:
            rc = lib.chitu_b200_qk_norm_rope_scatter(*common, _lib.ptr_array(out_ptrs), len(out_ptrs),
                                                     _DTYPES[out_dtype], *tail)
        else:
            rc = lib.chitu_b200_qk_norm_rope(*common, out.data_ptr(), _DTYPES[out.dtype], *tail)
    _lib.check(rc, "qk_norm_rope")
    _launched()
    return out


def qk_norm_rope_batch(
    jobs: Sequence[dict],
    num_heads: int,
    eps: float,
    rope_table: Optional[torch.Tensor],
    grid: Sequence[int] = (0, 0, 0),
    axis_split: Sequence[int] = (0, 0),
    pos_offset: int = 0,
    out_strides: Optional[Sequence[int]] = None,
    heads_per_group: Optional[int] = None,
    out_dtype: torch.dtype = torch.bfloat16,
    round_mid: bool = True,
    sync=None,
    stage_only: bool = False,
):
    """Up to three pre-attention jobs (q, k, v) in one launch; see ``chitu_b200_qk_norm_rope_batch``.

    With ``sync`` (a ``_lib.peer_sync_desc`` pair) the launch ends by announcing this rank's rows to its
    peers (``chitu_b200_qk_norm_rope_batch_signal``); with ``stage_only`` as well it only advances the layer
    epoch - its destinations are local, the attention launch's copy CTAs deliver and announce the rows
    (``chitu_b200_qk_norm_rope_batch_stage``).

    Each job is a dict with ``x [B,S,H*D]``, optional ``weight``, ``norm_mode``, ``rope_mode`` and
    either ``out`` (tensor), ``out_ptrs`` (list of device addresses) or neither (a contiguous
    ``[B,S,H,D]`` result is allocated).  All jobs share dtype, shape and placement.  Returns the list
    of output tensors (``None`` for jobs written through ``out_ptrs``).
    """
    x0 = jobs[0]["x"]
    B, S, C = x0.shape
    D = C // num_heads
    arr = (_lib.NormRopeJob * len(jobs))()
    keep, outs = [], []
    w_dtype = None
    for i, jb in enumerate(jobs):
        x = jb["x"]
        _require_cuda(x, jb.get("weight"), jb.get("out"))
        if x.shape != x0.shape or x.dtype != x0.dtype:
            raise ValueError("batched pre-attention jobs must share shape and dtype")
        if x.stride(2) != 1 or (B > 1 and x.stride(0) != S * x.stride(1)):
            x = x.contiguous()
        w = jb.get("weight")
        if w is not None:
            w = w.contiguous()
            if w_dtype is not None and w.dtype != w_dtype:
                raise ValueError("batched pre-attention jobs must share the weight dtype")
            w_dtype = w.dtype
        out, ptrs, rstd = jb.get("out"), jb.get("out_ptrs"), jb.get("rstd_out")
        if rstd is not None:
            if rstd.dtype != torch.float32 or rstd.numel() != B * S or not rstd.is_contiguous():
                raise ValueError("rstd_out must be a contiguous fp32 tensor of B*S elements")
            out = ptrs = None
            keep.append(rstd)
        arr[i].rstd_out = rstd.data_ptr() if rstd is not None else None
        if ptrs is None and out is None and rstd is None:
            if out_strides is not None:
                raise ValueError("explicit out_strides need out or out_ptrs in every job")
            out = torch.empty((B, S, num_heads, D), dtype=out_dtype, device=x.device)
        keep += [x, w, out]
        arr[i].x = x.data_ptr()
        arr[i].x_row_stride = x.stride(1)
        arr[i].weight = w.data_ptr() if w is not None else None
        arr[i].norm_mode = int(jb.get("norm_mode", 2))
        arr[i].rope_mode = int(jb.get("rope_mode", 0))
        arr[i].out = out.data_ptr() if out is not None else None
        if ptrs is not None:
            pa = _lib.ptr_array(ptrs)
            keep.append(pa)
            arr[i].out_ptrs = ctypes.cast(pa, ctypes.POINTER(ctypes.c_void_p))
            arr[i].n_out_ptrs = len(ptrs)
        else:
            arr[i].n_out_ptrs = 0
        outs.append(out)
    if out_strides is None:
        out_strides, heads_per_group = (S * C, C, 0, D), num_heads
    if rope_table is not None and (rope_table.dtype != torch.float32 or not rope_table.is_contiguous()):
        raise ValueError("rope_table must be a contiguous fp32 [rows, D/2, 2] tensor")
    split = (ctypes.c_int * 2)(int(axis_split[0]), int(axis_split[1]))
    lib = _lib.load()
    args = (
        arr, len(jobs), _DTYPES[x0.dtype], _DTYPES[w_dtype] if w_dtype is not None else _lib.DTYPE_FP32,
        float(eps), rope_table.data_ptr() if rope_table is not None else None,
        int(rope_table.shape[0]) if rope_table is not None else 0, int(grid[0]), int(grid[1]), int(grid[2]),
        split, int(pos_offset), _DTYPES[out_dtype], _lib.i64_array(out_strides), int(heads_per_group),
        B, S, num_heads, D, 1 if round_mid else 0,
    )
    with _on(x0.device):
        if sync is not None:
            fn = lib.chitu_b200_qk_norm_rope_batch_stage if stage_only else lib.chitu_b200_qk_norm_rope_batch_signal
            rc = fn(*args, ctypes.byref(sync[0]), _stream_ptr(x0.device))
        else:
            rc = lib.chitu_b200_qk_norm_rope_batch(*args, _stream_ptr(x0.device))
    _lib.check(rc, "qk_norm_rope_batch")
    _launched()
    return outs


def strided_copy(src: torch.Tensor, dst: torch.Tensor) -> torch.Tensor:
    """Copy a 5-d view ``src [n0,n1,n2,n3,row]`` (last dim contiguous) into contiguous ``dst``."""
    _require_cuda(src, dst)
    if src.dim() != 5 or dst.shape != src.shape or not dst.is_contiguous() or src.stride(4) != 1:
        raise ValueError("strided_copy: src must be 5-d with a contiguous last dim, dst contiguous of the same shape")
    es = src.element_size()
    lib = _lib.load()
    with _on(src.device):
        rc = lib.chitu_b200_strided_copy(
            src.data_ptr(), dst.data_ptr(), *[int(n) for n in src.shape[:4]], int(src.shape[4]) * es,
            _lib.i64_array([s * es for s in src.stride()[:4]]), _stream_ptr(src.device),
        )
    _lib.check(rc, "strided_copy")
    _launched()
    return dst


def layernorm_modulate(x: torch.Tensor, mul: Optional[torch.Tensor] = None, add: Optional[torch.Tensor] = None,
                       add_one: bool = False, eps: float = 1e-6, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``LayerNorm(x) * m + a`` for ``x [B, L, C]`` (fp32 or 16-bit); ``mul`` / ``add`` are ``[C]``, ``[1, C]``-like or ``[B, C]``-like
    fp32 (``m = 1 + mul`` with ``add_one``); see ``chitu_b200_layernorm_modulate``."""
    _require_cuda(x)
    if x.dtype not in _DTYPES or x.dim() != 3 or not x.is_contiguous():
        raise ValueError("layernorm_modulate: x must be a contiguous [B, L, C] tensor (fp32, bf16 or fp16)")
    B, L, C = x.shape

    def vec(t):
        if t is None:
            return None, 0
        t = t.reshape(-1, C)
        if t.dtype != torch.float32 or t.shape[0] not in (1, B) or t.stride(1) != 1:
            raise ValueError("layernorm_modulate: mul / add must be fp32 with C channels for 1 or B batches")
        return t, (t.stride(0) if t.shape[0] == B and B > 1 else 0)

    (m, ms), (a, as_) = vec(mul), vec(add)
    out = torch.empty((B, L, C), dtype=out_dtype, device=x.device)
    lib = _lib.load()
    with _on(x.device):
        rc = lib.chitu_b200_layernorm_modulate(
            x.data_ptr(), _DTYPES[x.dtype], out.data_ptr(), _DTYPES[out_dtype], B * L, L, C,
            m.data_ptr() if m is not None else None, ms,
            a.data_ptr() if a is not None else None, as_, int(add_one), float(eps), _stream_ptr(x.device))
    _lib.check(rc, "layernorm_modulate")
    _launched()
    return out


def gate_residual(x: torch.Tensor, y: torch.Tensor, gate: Optional[torch.Tensor] = None) -> torch.Tensor:
    """In place ``x += y * gate`` (``x [B, L, C]`` fp32 or 16-bit, ``y`` 16-bit, ``gate`` fp32 per batch and channel or None)."""
    _require_cuda(x, y)
    if x.dtype not in _DTYPES or x.dim() != 3 or not x.is_contiguous() or y.shape != x.shape or not y.is_contiguous():
        raise ValueError("gate_residual: x must be contiguous [B, L, C] and y contiguous of the same shape")
    B, L, C = x.shape
    g, gs = None, 0
    if gate is not None:
        g = gate.reshape(-1, C)
        if g.dtype != torch.float32 or g.shape[0] not in (1, B) or g.stride(1) != 1:
            raise ValueError("gate_residual: gate must be fp32 with C channels for 1 or B batches")
        gs = g.stride(0) if g.shape[0] == B and B > 1 else 0
    lib = _lib.load()
    with _on(x.device):
        rc = lib.chitu_b200_gate_residual(x.data_ptr(), _DTYPES[x.dtype], y.data_ptr(), _DTYPES[y.dtype], B * L, L, C,
                                          g.data_ptr() if g is not None else None, gs, _stream_ptr(x.device))
    _lib.check(rc, "gate_residual")
    _launched()
    return x


def cfg_combine(cond: torch.Tensor, uncond: torch.Tensor, scale: float, rescale: bool = False) -> torch.Tensor:
    """``uncond + scale * (cond - uncond)``, with ``rescale`` multiplied row-wise by ``||cond|| / ||result||`` over the last dim."""
    _require_cuda(cond, uncond)
    if cond.shape != uncond.shape or cond.dtype != uncond.dtype or cond.dtype not in _DTYPES:
        raise ValueError("cfg_combine: cond and uncond must share shape and dtype (bf16, fp16 or fp32)")
    cond, uncond = cond.contiguous(), uncond.contiguous()
    out = torch.empty_like(cond)
    C = cond.shape[-1]
    lib = _lib.load()
    with _on(cond.device):
        rc = lib.chitu_b200_cfg_combine(cond.data_ptr(), uncond.data_ptr(), out.data_ptr(), _DTYPES[cond.dtype],
                                        cond.numel() // C, C, float(scale), int(rescale), _stream_ptr(cond.device))
    _lib.check(rc, "cfg_combine")
    _launched()
    return out


def peer_copy_2d(dst_ptr: int, dst_pitch: int, src_ptr: int, src_pitch: int, width: int, rows: int,
                 device: torch.device) -> None:
    """``rows`` pieces of ``width`` bytes between device buffers (either may be peer-mapped), on the copy engines."""
    lib = _lib.load()
    with _on(device):
        rc = lib.chitu_b200_peer_copy_2d(int(dst_ptr), int(dst_pitch), int(src_ptr), int(src_pitch), int(width),
                                         int(rows), _stream_ptr(device))
    _lib.check(rc, "peer_copy_2d")


def scatter_rows(src: torch.Tensor, dst_ptrs: Sequence[int], rows: int, dst_batch_stride_bytes: int,
                 dst_row_stride_bytes: int) -> None:
    """``src [B, n_dest*rows, ...]`` contiguous: row ``(b, i*rows + j)`` goes to ``dst_ptrs[i] + b*batch + j*row`` bytes."""
    _require_cuda(src)
    if not src.is_contiguous() or src.dim() < 3 or src.shape[1] != rows * len(dst_ptrs):
        raise ValueError("scatter_rows: src must be contiguous [B, n_dest*rows, ...]")
    row_bytes = src[0, 0].numel() * src.element_size()
    lib = _lib.load()
    with _on(src.device):
        rc = lib.chitu_b200_scatter_rows(src.data_ptr(), _lib.ptr_array(dst_ptrs), len(dst_ptrs), int(src.shape[0]),
                                         int(rows), int(row_bytes), int(dst_batch_stride_bytes),
                                         int(dst_row_stride_bytes), _stream_ptr(src.device))
    _lib.check(rc, "scatter_rows")
    _launched()


def attn_fwd_scatter(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    out_ptrs: Sequence[int],
    rows_per_dest: int,
    dest_batch_stride: int,
    dest_row_stride: int,
    dest_head_offset: int,
    softmax_scale: Optional[float] = None,
    n_splits: Optional[int] = None,
    workspace: Optional[torch.Tensor] = None,
) -> None:
    """Attention whose query row ``r`` is stored to ``out_ptrs[r // rows_per_dest]``; see ``chitu_b200_attn_fwd_scatter``."""
    _require_cuda(q, k, v)
    B, Sq, H, D = q.shape
    Sk = k.shape[1]
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise NotImplementedError("attention kernel takes bf16 or fp16 q/k/v of one dtype")
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(D)
    lib = _lib.load()
    if n_splits is None:
        n_splits = auto_key_splits(B, Sq, Sk, H)
    ws_ptr, ws_bytes = None, 0
    if n_splits > 1:
        need = int(lib.chitu_b200_attn_splitkv_workspace_bytes(B, Sq, H, D, n_splits))
        ws = workspace if workspace is not None else _split_scratch(q.device, need)
        if ws.numel() * ws.element_size() < need or ws.device != q.device:
            raise ValueError(f"attn_fwd_scatter: workspace must hold {need} bytes on {q.device}")
        ws_ptr, ws_bytes = ws.data_ptr(), ws.numel()
    with _on(q.device):
        rc = lib.chitu_b200_attn_fwd_scatter(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _lib.ptr_array(out_ptrs), len(out_ptrs), int(rows_per_dest),
            int(dest_batch_stride), int(dest_row_stride), int(dest_head_offset), None, B, Sq, Sk, H, D,
            _lib.i64_array(q.stride()), _lib.i64_array(k.stride()), _lib.i64_array(v.stride()), scale,
            _DTYPES[q.dtype], int(n_splits), ws_ptr, ws_bytes, status_word(q.device).data_ptr(),
            _stream_ptr(q.device),
        )
    _lib.check(rc, "attn_fwd_scatter")
    _launched(1)


def peer_barrier(flag_ptrs: Sequence[int], rank: int, world: int, device: torch.device) -> None:
    """Enqueue the bounded cross-GPU barrier on the current stream; see ``chitu_b200_peer_barrier``."""
    lib = _lib.load()
    with _on(device):
        rc = lib.chitu_b200_peer_barrier(_lib.ptr_array(flag_ptrs), int(rank), int(world),
                                         status_word(device).data_ptr(), _stream_ptr(device))
    _lib.check(rc, "peer_barrier")
    _launched()


def attn_fwd_exchange(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    out_ptrs: Sequence[int],
    rows_per_dest: int,
    dest_batch_stride: int,
    dest_row_stride: int,
    dest_head_offset: int,
    rows_per_src: int,
    sync,
    softmax_scale: Optional[float] = None,
    n_splits: Optional[int] = None,
    workspace: Optional[torch.Tensor] = None,
    prefix_rows: int = 0,
    prefix_ptrs: Optional[Sequence[int]] = None,
    prefix_batch_stride: int = 0,
    prefix_row_stride: int = 0,
    prefix_head_offset: int = 0,
    push=None,
) -> None:
    """:func:`attn_fwd_scatter` over exchange buffers guarded by arrival flags; see ``chitu_b200_attn_fwd_exchange``.
    With ``push`` (a ``_lib.push_desc`` pair) the launch also delivers the staged rows to the peers
    (``chitu_b200_attn_fwd_exchange_push``)."""
    _require_cuda(q, k, v)
    B, Sq, H, D = q.shape
    Sk = k.shape[1]
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise NotImplementedError("attention kernel takes bf16 or fp16 q/k/v of one dtype")
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(D)
    lib = _lib.load()
    if n_splits is None:
        n_splits = auto_key_splits(B, Sq, Sk, H)
    ws_ptr, ws_bytes = None, 0
    if n_splits > 1:
        need = int(lib.chitu_b200_attn_splitkv_workspace_bytes(B, Sq, H, D, n_splits))
        ws = workspace if workspace is not None else _split_scratch(q.device, need)
        if ws.numel() * ws.element_size() < need or ws.device != q.device:
            raise ValueError(f"attn_fwd_exchange: workspace must hold {need} bytes on {q.device}")
        ws_ptr, ws_bytes = ws.data_ptr(), ws.numel()
    if push is not None:
        if prefix_rows:
            raise NotImplementedError("push mode has no replicated prefix")
        with _on(q.device):
            rc = lib.chitu_b200_attn_fwd_exchange_push(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), _lib.ptr_array(out_ptrs), len(out_ptrs),
                int(rows_per_dest), int(dest_batch_stride), int(dest_row_stride), int(dest_head_offset), B, Sq, Sk, H,
                D, _lib.i64_array(q.stride()), _lib.i64_array(k.stride()), _lib.i64_array(v.stride()), scale,
                _DTYPES[q.dtype], int(n_splits), ws_ptr, ws_bytes, int(rows_per_src), ctypes.byref(push[0]),
                ctypes.byref(sync[0]), status_word(q.device).data_ptr(), _stream_ptr(q.device),
            )
        _lib.check(rc, "attn_fwd_exchange_push")
        _launched(1)
        return
    with _on(q.device):
        rc = lib.chitu_b200_attn_fwd_exchange(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _lib.ptr_array(out_ptrs), len(out_ptrs), int(rows_per_dest),
            int(dest_batch_stride), int(dest_row_stride), int(dest_head_offset), B, Sq, Sk, H, D,
            _lib.i64_array(q.stride()), _lib.i64_array(k.stride()), _lib.i64_array(v.stride()), scale,
            _DTYPES[q.dtype], int(n_splits), ws_ptr, ws_bytes, int(rows_per_src), int(prefix_rows),
            _lib.ptr_array(prefix_ptrs) if prefix_ptrs else None, int(prefix_batch_stride), int(prefix_row_stride),
            int(prefix_head_offset), ctypes.byref(sync[0]),
            status_word(q.device).data_ptr(), _stream_ptr(q.device),
        )
    _lib.check(rc, "attn_fwd_exchange")
    _launched(1)


def set_cluster_merge(enable: bool) -> bool:
    """Merge two key ranges through a thread-block cluster's shared memory (default) or through the workspace;
    returns the previous setting.  ``CHITU_B200_CLUSTER_MERGE=0`` at import time selects the workspace form."""
    return bool(_lib.load().chitu_b200_set_cluster_merge(1 if enable else 0))


def stamp(slots: torch.Tensor, index: int) -> None:
    """Enqueue a launch that writes the GPU's nanosecond timer into ``slots[index]`` (int64 tensor on the GPU);
    works inside a captured graph.  Not counted as a launch of the hot path."""
    if slots.dtype != torch.int64 or not slots.is_cuda or not slots.is_contiguous():
        raise ValueError("stamp: slots must be a contiguous int64 CUDA tensor")
    if not 0 <= index < slots.numel():
        raise IndexError("stamp: index out of range")
    with _on(slots.device):
        rc = _lib.load().chitu_b200_stamp(slots.data_ptr() + 8 * int(index), _stream_ptr(slots.device))
    _lib.check(rc, "stamp")


def push_ctas(B: int, Sq: int, H: int, n_splits: int) -> int:
    """Copy CTAs that push mode would add to an attention launch of this shape on the current device (0: none)."""
    return int(_lib.load().chitu_b200_push_ctas(int(B), int(Sq), int(H), int(n_splits)))


def peer_wait_outputs(sync, device: torch.device) -> None:
    """Enqueue the bounded wait for every rank's output flag; see ``chitu_b200_peer_wait_outputs``."""
    lib = _lib.load()
    with _on(device):
        rc = lib.chitu_b200_peer_wait_outputs(ctypes.byref(sync[0]), status_word(device).data_ptr(), _stream_ptr(device))
    _lib.check(rc, "peer_wait_outputs")
    _launched()


# ---------------------------------------------------------------------------------------------- paged key/value cache
# Calls of a generation loop wait for the host: tensors are asked for each attribute once, arrays go down as packed bytes.
_CACHE_HEAD_DIM = 128
_CACHE_PAGES = (16, 32, 64, 128, 256)
_APPEND_FEW = 4  # appended tokens of the longest sequence up to which the library takes its form for single tokens
_POSITION_DTYPES = (torch.int32, torch.int64)


def _token_rows(t: torch.Tensor) -> torch.Tensor:
    """``t [tokens, heads, D]`` as the kernels take it: channels contiguous, 16-byte aligned, otherwise of any strides."""
    s0, s1, s2 = t.stride()
    if s2 == 1 and s0 and s1 and not (s0 | s1) * t.element_size() & 15 and not t.data_ptr() & 15:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _check_rope(rope_table: torch.Tensor, head_dim: int, what: str) -> int:
    """Rotated channels of a table of (cos, sin) pairs ``[rows, rot / 2, 2]``."""
    shape = rope_table.shape
    if rope_table.dtype != torch.float32 or len(shape) != 3 or shape[2] != 2 or not rope_table.is_contiguous():
        raise ValueError(f"{what}: rope_table must be a contiguous fp32 [rows, rot / 2, 2] tensor")
    rot = 2 * shape[1]
    if rot > head_dim:
        raise ValueError(f"{what}: rope_table turns {rot} channels, a head has {head_dim}")
    if rot % 16 or rot == 0:
        raise NotImplementedError(f"{what}: rotated channels must be a positive multiple of 16 (got {rot})")
    return rot


def _check_positions(positions: torch.Tensor, tokens: int, what: str) -> torch.Tensor:
    if positions.dtype not in _POSITION_DTYPES or positions.numel() != tokens:
        raise ValueError(f"{what}: positions must be int32 or int64, one per token ({tokens})")
    return positions if positions.is_contiguous() else positions.contiguous()


def rotary(x, positions: torch.Tensor, rope_table: torch.Tensor, interleaved: bool = True, out=None):
    """Rotary embedding of one tensor ``[T, H, D]`` or of up to three of the same tokens (``[q, k]``) in one launch.

    The first ``rot = 2 * rope_table.shape[1]`` channels of every head turn by row ``positions[t]`` of ``rope_table`` (fp32
    (cos, sin) pairs ``[rows, rot / 2, 2]``; see ``pre_attention.scaled_rope_table``); the others pass, and so do tokens whose
    position is outside the table.  Pairs are adjacent channels, as everywhere in this library, or with
    ``interleaved=False`` channels ``(j, j + rot / 2)``.  bf16, fp16 or fp32 in and out; ``D`` and ``rot`` multiples of 16.
    ``out`` (a tensor, or one per tensor of the list) may be ``x`` itself, each in its own place; other overlaps are refused as
    far as they begin at one address.  ``[B, S, H, D]`` tensors are taken as ``B * S`` tokens.
    See ``chitu_b200_rotary``.
    """
    single = isinstance(x, torch.Tensor)
    xs = (x,) if single else tuple(x)
    n = len(xs)
    outs = (None,) * n if out is None else (out,) if single else tuple(out)
    if not 1 <= n <= 3 or len(outs) != n:
        raise ValueError("rotary: one to three tensors, and as many outputs")
    first = xs[0]
    shape, dtype = first.shape, first.dtype
    dim = len(shape)
    if dim not in (3, 4) or dtype not in _DTYPES:
        raise ValueError("rotary: x must be [T, H, D] or [B, S, H, D], bf16, fp16 or fp32")
    lead, D, on = shape[:-2], shape[-1], first.get_device()
    n_tokens = shape[0] if dim == 3 else shape[0] * shape[1]
    if D % 16 or D > 512:
        raise NotImplementedError(f"rotary: head_dim must be a multiple of 16 up to 512 (got {D})")
    rot = _check_rope(rope_table, D, "rotary")
    positions = _check_positions(positions, n_tokens, "rotary")
    ptrs, out_ptrs, strides, out_strides, heads, keep, results = [], [], [], [], [], [], []
    for t, o in zip(xs, outs):
        s = t.shape
        if s[:-2] != lead or s[-1] != D or t.dtype != dtype or t.get_device() != on:
            raise ValueError("rotary: tensors of one call share tokens, head_dim, dtype and device")
        if s[-2] == 0:
            raise ValueError("rotary: a tensor has no heads")
        rows = _token_rows(t if dim == 3 else t.flatten(0, 1))
        if o is None:
            o = torch.empty_like(t, memory_format=torch.contiguous_format)
            out_ptrs.append(o.data_ptr())
            out_strides += (s[-2] * D, D)
        else:
            if o.shape != s or o.dtype != dtype or o.get_device() != on:
                raise ValueError("rotary: out must have x's shape, dtype and device")
            o_rows = o if dim == 3 else o.flatten(0, 1)
            if o_rows.data_ptr() != o.data_ptr() or _token_rows(o_rows) is not o_rows:
                raise ValueError("rotary: out must have contiguous channels and 16-byte aligned rows")
            out_ptrs.append(o.data_ptr())
            out_strides += o_rows.stride()[:2]
        ptrs.append(rows.data_ptr())
        strides += rows.stride()[:2]
        heads.append(s[-2])
        keep.append(rows)
        results.append(o)
    if out is not None and n_tokens:
        for i, at in enumerate(out_ptrs):
            if at in out_ptrs[:i] or any(at == p and (i != j or strides[2 * i:2 * i + 2] != out_strides[2 * i:2 * i + 2]) for j, p in enumerate(ptrs)):
                raise ValueError("rotary: an output may only take the place of its own input, with its strides")
    if on < 0:
        _require_cuda(first)
    if positions.get_device() != on or rope_table.get_device() != on:
        raise ValueError("rotary: positions and rope_table must be on x's device")
    if n_tokens == 0:
        return results[0] if single else results
    args = (_lib.PTRS[n](*ptrs), _lib.PTRS[n](*out_ptrs), _lib.I64S[2 * n](*strides), _lib.I64S[2 * n](*out_strides), _lib.INTS[n](*heads),
            n, n_tokens, D, rot, _DTYPES[dtype], positions.data_ptr(), positions.dtype == torch.int64, rope_table.data_ptr(),
            rope_table.shape[0], bool(interleaved), torch._C._cuda_getCurrentRawStream(on))
    if torch._C._cuda_getDevice() == on:
        rc = _lib.load().chitu_b200_rotary(*args)
    else:
        with torch.cuda.device(on):
            rc = _lib.load().chitu_b200_rotary(*args)
    if rc:
        _lib.check(rc, "rotary")
    _launched()
    return results[0] if single else results


def _pack_cache(k_cache, v_cache, block_table, kv_lens, cu_seqlens, k_scale, v_scale, dtype, what):
    """``chitu_b200_kv_cache`` of a call as bytes, after the checks that need no GPU: ``(bytes, batch, table width, page_size, heads)``."""
    shape, cache_dtype = k_cache.shape, k_cache.dtype
    if len(shape) != 4 or v_cache.shape != shape or v_cache.dtype != cache_dtype:
        raise ValueError(f"{what}: k_cache and v_cache must be [pages, page_size, H, 128] of one shape and dtype")
    n_pages, page, heads, D = shape
    if D != _CACHE_HEAD_DIM:
        raise NotImplementedError(f"{what}: head_dim must be {_CACHE_HEAD_DIM} (got {D})")
    if page not in _CACHE_PAGES:
        raise NotImplementedError(f"{what}: page_size must be one of {_CACHE_PAGES} (got {page})")
    if n_pages == 0 or heads == 0:
        raise ValueError(f"{what}: the cache has no pages or no heads")
    eight = cache_dtype == torch.float8_e4m3fn
    if not eight and cache_dtype != dtype:
        raise NotImplementedError(f"{what}: pages hold float8_e4m3fn or the inputs' type {dtype} (got {cache_dtype})")
    on = k_cache.get_device()
    kp, vp = k_cache.data_ptr(), v_cache.data_ptr()
    k0, k1, k2, k3 = k_cache.stride()
    v0, v1, v2, v3 = v_cache.stride()
    if k3 != 1 or v3 != 1 or not (k0 and k1 and k2 and v0 and v1 and v2) or (k0 | k1 | k2 | v0 | v1 | v2) & (15 if eight else 7) or (kp | vp) & 15:
        raise ValueError(f"{what}: cache channels must be contiguous, rows and pages 16-byte aligned")
    if eight:
        for s in (k_scale, v_scale):
            if s is None or s.dtype != torch.float32 or s.shape != (n_pages, heads) or s.get_device() != on:
                raise ValueError(f"{what}: 8-bit pages need fp32 k_scale and v_scale [pages, H] = ({n_pages}, {heads})")
        (ks0, ks1), (vs0, vs1), ksp, vsp = k_scale.stride(), v_scale.stride(), k_scale.data_ptr(), v_scale.data_ptr()
    else:
        if k_scale is not None or v_scale is not None:
            raise ValueError(f"{what}: 16-bit pages have no scales")
        ks0 = ks1 = vs0 = vs1 = ksp = vsp = 0
    shape = block_table.shape
    if len(shape) != 2 or block_table.dtype != torch.int32 or shape[1] == 0 or block_table.stride(1) != 1:
        raise ValueError(f"{what}: block_table must be an int32 [B, pages] tensor with contiguous rows")
    B, width = shape
    if kv_lens.dtype != torch.int32 or kv_lens.shape != (B,) or not kv_lens.is_contiguous():
        raise ValueError(f"{what}: kv_lens must be a contiguous int32 [B] tensor (B = {B})")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.shape != (B + 1,) or not cu_seqlens.is_contiguous():
        raise ValueError(f"{what}: cu_seqlens must be a contiguous int32 [B + 1] tensor (B = {B})")
    if v_cache.get_device() != on or block_table.get_device() != on or kv_lens.get_device() != on or cu_seqlens.get_device() != on:
        raise ValueError(f"{what}: the cache, its table and its lengths must be on one device")
    packed = _lib.KV_CACHE.pack(kp, vp, ksp, vsp, k0, k1, k2, v0, v1, v2, ks0, ks1, vs0, vs1, block_table.data_ptr(), kv_lens.data_ptr(),
                                cu_seqlens.data_ptr(), block_table.stride(0), B, width, n_pages, page, heads,
                                _lib.CACHE_E4M3 if eight else _lib.CACHE_16BIT)
    return packed, B, width, page, heads


def _check_tokens(t: torch.Tensor, name: str, what: str):
    """Shape and type of packed tokens."""
    shape, dtype = t.shape, t.dtype
    if len(shape) != 3 or shape[2] != _CACHE_HEAD_DIM:
        raise ValueError(f"{what}: {name} must be packed tokens [T, H, {_CACHE_HEAD_DIM}]")
    if dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f"{what}: {name} must be bf16 or fp16")
    return shape, dtype


def _expected_new(tokens: int, batch: int) -> int:
    """``max_new`` of an append that does not say: with a token at least of every sequence the longest brings ``longest`` at most, and
    up to ``_APPEND_FEW`` of them suit the form that walks them one after the other.  A prompt may not go there unseen: 2000 tokens
    beside 699 single ones, 8-bit pages, take 2415 us there and 255 in the other form, which costs 64 sequences of two tokens 14 us for 5."""
    longest = tokens - batch + 1
    return max(1, longest) if longest <= _APPEND_FEW else max(_APPEND_FEW + 1, -(-tokens // batch))


def kv_cache_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    kv_lens: torch.Tensor,
    cu_seqlens: torch.Tensor,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    rope_table: Optional[torch.Tensor] = None,
    interleaved: bool = True,
    q: Optional[torch.Tensor] = None,
    max_new: Optional[int] = None,
) -> Optional[torch.Tensor]:
    """Append packed tokens ``k, v [T, H, 128]`` to a paged cache, keys rotated on the way; see ``chitu_b200_kv_append``.

    ``k_cache, v_cache [pages, page_size, H, 128]`` hold the inputs' 16-bit type, or float8_e4m3fn codes with fp32 scales
    ``k_scale, v_scale [pages, H]``; tokens or heads may be outermost in memory.  ``block_table [B, n]`` (int32) names the pages of a
    sequence in order, ``kv_lens [B]`` (int32) counts its tokens WITH the new ones, ``cu_seqlens [B + 1]`` (int32) says
    which rows of ``k`` and ``v`` are its: token ``i`` of the ``n_b`` new ones takes position ``kv_lens[b] - n_b + i``.  Rows behind
    the last sequence are left alone.

    With ``rope_table`` keys turn by the row of their position, or of ``positions [T]`` where given (a clip's per-token rows), and
    ``q [T, Hq, 128]``, if given, is rotated by the same launch and returned (rows behind the last sequence are not written).

    ``max_new`` is how many tokens the longest sequence brings; it chooses the kernel and sizes the launch, results do not depend on it.  By
    default it is taken that every sequence brings a token.  State it where that is far off: a batch in which few sequences bring
    anything takes a microsecond for each token of the longest one otherwise, one of two to four tokens each the form for prompts.
    """
    what = "kv_cache_append"
    shape, dtype = _check_tokens(k, "k", what)
    if v.shape != shape or v.dtype != dtype:
        raise ValueError(f"{what}: shape mismatch: k {tuple(k.shape)}, v {tuple(v.shape)}")
    packed, B, _, page, heads = _pack_cache(k_cache, v_cache, block_table, kv_lens, cu_seqlens, k_scale, v_scale, dtype, what)
    T = shape[0]
    if shape[1] != heads:
        raise ValueError(f"{what}: k has {shape[1]} heads, the cache {heads}")
    if k_scale is not None and (0 in k_scale.stride() or 0 in v_scale.stride()):
        raise ValueError(f"{what}: every page and head needs a scale of its own to write")
    on = k.get_device()
    q_heads = 0
    if q is not None:
        q_shape, q_dtype = _check_tokens(q, "q", what)
        q_heads = q_shape[1]
        if q_shape[0] != T or q_dtype != dtype or q_heads == 0:
            raise ValueError(f"{what}: q must be [T, Hq, 128] of k's tokens and dtype")
        if rope_table is None:
            raise ValueError(f"{what}: q is taken to be rotated, which needs a rope_table")
    rot = rows = table_ptr = 0
    if rope_table is not None:
        rot, rows, table_ptr = _check_rope(rope_table, _CACHE_HEAD_DIM, what), rope_table.shape[0], rope_table.data_ptr()
    elif positions is not None:
        raise ValueError(f"{what}: positions without a rope_table")
    if positions is not None:
        positions = _check_positions(positions, T, what)
    if on < 0:
        _require_cuda(k)
    for t in (v, k_cache, q, positions, rope_table):
        if t is not None and t.get_device() != on:
            raise ValueError(f"{what}: all tensors must be on one device")
    k, v = _token_rows(k), _token_rows(v)
    i64x2 = _lib.I64S[2]
    q_out = q_ptr = q_strides = q_out_ptr = None
    if q is not None:
        q = _token_rows(q)
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        q_ptr, q_strides, q_out_ptr = q.data_ptr(), i64x2(*q.stride()[:2]), q_out.data_ptr()
    if T == 0 or B == 0:
        return q_out
    if max_new is None:
        max_new = _expected_new(T, B)
    args = (packed, k.data_ptr(), v.data_ptr(), q_ptr, i64x2(*k.stride()[:2]), i64x2(*v.stride()[:2]), q_strides, q_out_ptr, q_heads, T,
            _DTYPES[dtype], int(max_new), None if positions is None else positions.data_ptr(),
            positions is not None and positions.dtype == torch.int64, table_ptr, rows, rot, bool(interleaved),
            torch._C._cuda_getCurrentRawStream(on))
    if torch._C._cuda_getDevice() == on:
        rc = _lib.load().chitu_b200_kv_append(*args)
    else:
        with torch.cuda.device(on):
            rc = _lib.load().chitu_b200_kv_append(*args)
    if rc:
        _lib.check(rc, what)
    # (8-bit pages of 256 tokens: keys and values in one launch, queries in another)
    _launched(2 if page == 256 and q is not None and k_scale is not None and min(int(max_new), T) > _APPEND_FEW else 1)
    return q_out


def _cache_scratch(device: torch.device, nbytes: int) -> torch.Tensor:
    """Scratch of one call: of an eager one that of the cuts (:func:`_cut_scratch`; a stream's calls follow one another, and both leave the
    counters at its head zero), of a captured one its own (:func:`_split_scratch`)."""
    with _on(device):
        if not torch.cuda.is_current_stream_capturing():
            return _cut_scratch(device, nbytes)
    return _split_scratch(device, nbytes)


@functools.lru_cache(maxsize=256)
def _cache_workspace_bytes(heads: int, q_heads: int, max_q: int) -> int:
    return int(_lib.load().chitu_b200_attn_cache_workspace_bytes(heads, q_heads, max_q))


def attn_fwd_cache(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    kv_lens: torch.Tensor,
    cu_seqlens: torch.Tensor,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    causal: bool = False,
    return_lse: bool = False,
    out: Optional[torch.Tensor] = None,
    max_q: Optional[int] = None,
    max_kv: Optional[int] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Attention of packed queries ``q [T, Hq, 128]`` over a paged cache of ``H`` key heads; see ``chitu_b200_attn_fwd_cache``.

    The cache, its table and its lengths are those of :func:`kv_cache_append` (call that first: ``kv_lens`` counts this call's
    tokens).  ``Hq`` is a multiple of ``H``.  A query of sequence ``b`` attends to all of its ``kv_lens[b]`` keys, with
    ``causal`` query ``i`` of ``n_b`` only to keys up to position ``kv_lens[b] - n_b + i``.  Returns
    ``(out [T, Hq, 128], lse [Hq, T] fp32 | None)``; a query without a visible key gives zeros and ``-inf``, rows behind the last
    sequence are left as they were in ``out``.  With ``lse[None]`` the result folds into others by :func:`lse_combine`.

    ``max_q`` and ``max_kv`` are how many queries and keys the longest sequence has (defaults: the average number of queries,
    what the table can hold); they choose the kernel and its grid, results are right whatever they are.  One kernel serves the
    whole call, so a prompt and many single tokens cost more together than apart (512 queries beside 63 single ones over
    16000 keys, 8 key heads: 848 us, in two calls 44 and 326).
    """
    what = "attn_fwd_cache"
    shape, dtype = _check_tokens(q, "q", what)
    packed, B, width, page, heads = _pack_cache(k_cache, v_cache, block_table, kv_lens, cu_seqlens, k_scale, v_scale, dtype, what)
    T, Hq, D = shape
    if Hq == 0 or Hq % heads:
        raise ValueError(f"{what}: {Hq} query heads over {heads} key heads")
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not 0.0 < scale < 1e30:
        raise ValueError(f"{what}: softmax_scale must be positive and finite (got {scale})")
    device, on = q.device, q.get_device()
    if out is not None and (out.shape != shape or out.dtype != dtype or not out.is_contiguous() or out.get_device() != on):
        raise ValueError(f"{what}: out must be a contiguous tensor of q's shape, dtype and device")
    if on < 0:
        _require_cuda(q)
    if k_cache.get_device() != on:
        raise ValueError(f"{what}: q and the cache must be on one device")
    q = _token_rows(q)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((Hq, T), dtype=torch.float32, device=device) if return_lse else None
    if T == 0 or B == 0:
        return out, lse
    max_q = -(-T // B) if max_q is None else max(1, int(max_q))
    max_kv = width * page if max_kv is None else max(1, min(int(max_kv), width * page))
    need = _cache_workspace_bytes(heads, Hq, max_q)
    ws = _cache_scratch(device, need)
    args = (packed, q.data_ptr(), _lib.I64S[2](*q.stride()[:2]), out.data_ptr(), None if lse is None else lse.data_ptr(), Hq, T, scale,
            bool(causal), _DTYPES[dtype], max_q, max_kv, ws.data_ptr(), ws.numel(), status_word(device).data_ptr(),
            torch._C._cuda_getCurrentRawStream(on))
    if torch._C._cuda_getDevice() == on:
        rc = _lib.load().chitu_b200_attn_fwd_cache(*args)
    else:
        with torch.cuda.device(on):
            rc = _lib.load().chitu_b200_attn_fwd_cache(*args)
    if rc:
        _lib.check(rc, what)
    # (chunks of queries: what the borders of the CTAs' runs have cut is joined by a kernel of its own)
    _launched(2 if max_q * (Hq // heads) > 32 and Hq // heads <= 128 else 1)
    return out, lse
