"""Drop-in replacements for tinyvllm's attention functions, on the sm_100a kernels.

``paged_decode_attention`` and ``flash_prefill_attention`` keep the signatures
and argument meaning of ``tinyvllm/model/llama.py:97-108`` and ``:58-63``;
the arguments are torch CUDA tensors instead of tinygrad Tensors.  Each call
goes straight to ``libtvk.so`` through ctypes with raw device pointers on the
current torch stream.
"""

from __future__ import annotations

import ctypes
import threading
from typing import Dict, Optional, Tuple

import torch

from . import _lib

_ws_lock = threading.Lock()
_workspaces: Dict[Tuple[int, int, str], torch.Tensor] = {}


def _workspace(device: torch.device, nbytes: int, kind: str = "decode") -> torch.Tensor:
    """Per-(device, stream, kernel family) scratch buffer, grown on demand and zeroed
    when created (its first word is the kernels' time-out status, which a larger buffer
    takes over)."""
    key = (device.index if device.index is not None else torch.cuda.current_device(),
           torch.cuda.current_stream(device).cuda_stream, kind)
    with _ws_lock:
        ws = _workspaces.get(key)
        if ws is None or ws.numel() < nbytes:
            grown = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
            if ws is not None:
                grown[:4].copy_(ws[:4])
            ws = _workspaces[key] = grown
        return ws


_capture_workspaces: Dict[tuple, Tuple[int, torch.Tensor]] = {}


def _capture_workspace(index: int, nbytes: int, kind: str, zero_tail: int) -> Optional[torch.Tensor]:
    """While device ``index``'s current stream records a CUDA graph: a workspace of that graph and stream
    alone, so that graphs recorded on one stream, and branches of one graph, may run at
    the same time.  Its header and last ``zero_tail`` bytes are zeroed by the graph itself
    at every replay; where a call needs a larger one than those before it, that takes over
    their status word.  It lies in the graph's memory pool and lives as long as that; here
    it is only kept until the stream's next recording.  None while nothing is recorded."""
    if index == torch.cuda.current_device() and not torch.cuda.is_current_stream_capturing():
        return None
    stream = _lib.raw_stream(index)
    if stream == 0:                      # a device's default stream cannot record
        return None
    capture = ctypes.c_ulonglong()
    rc = _lib.lib().tvk_stream_capture_id(ctypes.byref(capture), stream)
    _lib.check(rc, "tvk_stream_capture_id")
    if capture.value == 0:               # another device's stream records, or none does
        return None
    key = (index, stream, kind)
    with _ws_lock:
        of, ws = _capture_workspaces.get(key, (0, None))
        if of != capture.value or ws.numel() < nbytes:
            before = ws if of == capture.value else None
            ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=torch.device("cuda", index))
            ws[:256].zero_()
            if before is not None:
                ws[:4].copy_(before[:4])
            if zero_tail:
                ws[nbytes - zero_tail:].zero_()
            _capture_workspaces[key] = (capture.value, ws)
        return ws


_q8_fixed_bytes = 0


def _workspace_q8(index: int, batch: int, n_kv_heads: int) -> torch.Tensor:
    """The workspace of an 8-bit decode call on the current stream of device ``index``."""
    global _q8_fixed_bytes
    L = _lib.lib()
    if not _q8_fixed_bytes:
        _q8_fixed_bytes = L.tvk_paged_decode_q8_workspace_size(0, 0)
    nbytes = L.tvk_paged_decode_q8_workspace_size(batch, n_kv_heads)
    return call_workspace(index, nbytes, "decode_q8", nbytes - _q8_fixed_bytes)


def call_workspace(index: int, nbytes: int, kind: str, zero_tail: int = 0) -> torch.Tensor:
    """A workspace of at least ``nbytes`` for a call on the current stream of device ``index``:
    the recorded graph's own, or the stream's (zeroed once)."""
    ws = _capture_workspace(index, nbytes, kind, zero_tail)
    if ws is None:
        ws = _workspaces.get((index, _lib.raw_stream(index), kind))
        if ws is None or ws.numel() < nbytes:
            ws = _workspace(torch.device("cuda", index), nbytes, kind)
    return ws


def workspace_status(device: Optional[torch.device] = None, kind: str = "decode") -> int:
    """Status word of the current stream's workspace (non-zero: a kernel wait timed out)."""
    device = device or torch.device("cuda", torch.cuda.current_device())
    ws = _workspace(device, 0, kind)
    return int(ws[:4].view(torch.int32).item())


def status_word(device: Optional[torch.device] = None, kind: str = "decode") -> torch.Tensor:
    """The current stream's workspace status word as a one-element int32 device tensor
    (a view: a CUDA graph can copy it out alongside its results)."""
    device = device or torch.device("cuda", torch.cuda.current_device())
    ws = None
    if kind == "decode_q8":
        index = device.index if device.index is not None else torch.cuda.current_device()
        ws = _capture_workspace(index, 0, kind, 0)
    return (_workspace(device, 0, kind) if ws is None else ws)[:4].view(torch.int32)


def check_workspace(device: Optional[torch.device] = None, kind: str = "decode", what: str = "kernel") -> None:
    """Raise ``TvkError`` if a bounded wait inside a kernel that used the current
    stream's ``kind`` workspace gave up (its output is then incomplete).  Reads the
    status word (a device-to-host copy, so the stream is synchronised); on a
    time-out the workspace header is zeroed first, so the next call starts clean."""
    device = device or torch.device("cuda", torch.cuda.current_device())
    ws = _workspace(device, 0, kind)
    if int(ws[:4].view(torch.int32).item()) != 0:
        ws[:256].zero_()
        raise _lib.TvkError(f"{what}: a bounded wait inside the kernel timed out; the output is incomplete")


def paged_decode_attention(queries: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           block_tables: torch.Tensor, context_lens: torch.Tensor,
                           n_heads: int, n_kv_heads: int, head_dim: int, block_size: int,
                           max_context_len: Optional[int] = None, *,
                           out: Optional[torch.Tensor] = None, check: bool = False) -> torch.Tensor:
    """Paged attention for decode (tinyvllm/model/llama.py:97-144).

    queries [B,1,Hq,D]; k_cache/v_cache [N,block_size,Hkv,D] (one layer's pool);
    block_tables int32 [B,max_blocks]; context_lens int32 [B].  Returns [B,1,Hq,D]
    in the pool dtype.  ``max_context_len=None`` attends over the whole table
    width masked by ``context_lens`` like the reference; an int truncates the
    table to ``ceil(max_context_len / block_size)`` blocks first.  ``check=True``
    synchronises the stream and raises ``TvkError`` if a bounded wait inside the
    kernel timed out (the call is otherwise asynchronous; the engine checks once
    per step instead).
    """
    dev = _lib.require_cuda(queries, k_cache, v_cache, block_tables, context_lens)
    B = queries.shape[0]
    if queries.shape[1:] != (1, n_heads, head_dim):
        raise ValueError(f"queries must be [B,1,{n_heads},{head_dim}], got {tuple(queries.shape)}")
    if k_cache.dim() != 4 or k_cache.shape[1:] != (block_size, n_kv_heads, head_dim) or v_cache.shape != k_cache.shape:
        raise ValueError(f"k_cache/v_cache must be [N,{block_size},{n_kv_heads},{head_dim}], got "
                         f"{tuple(k_cache.shape)} / {tuple(v_cache.shape)}")
    if queries.dtype != k_cache.dtype or v_cache.dtype != k_cache.dtype:
        raise TypeError("queries, k_cache and v_cache must share one dtype")
    if block_tables.dtype != torch.int32 or context_lens.dtype != torch.int32:
        raise TypeError("block_tables and context_lens must be int32")
    if block_tables.dim() != 2 or block_tables.shape[0] != B or context_lens.shape != (B,):
        raise ValueError("block_tables must be [B,max_blocks] and context_lens [B]")
    for name, t in (("queries", queries), ("k_cache", k_cache), ("v_cache", v_cache),
                    ("block_tables", block_tables), ("context_lens", context_lens)):
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    if out is None:
        out = torch.empty_like(queries)
    max_blocks = block_tables.shape[1]
    mcl = -1 if max_context_len is None else int(max_context_len)
    L = _lib.lib()
    nbytes = L.tvk_paged_decode_workspace_size(B, n_heads, n_kv_heads, head_dim, block_size, max_blocks, mcl)
    ws = _workspace(dev, nbytes)
    rc = L.tvk_paged_decode_attention(
        _lib.ptr(queries), _lib.ptr(k_cache), _lib.ptr(v_cache), _lib.ptr(block_tables),
        _lib.ptr(context_lens), _lib.ptr(out),
        B, n_heads, n_kv_heads, head_dim, block_size, k_cache.shape[0], max_blocks, mcl,
        _lib.dtype_code(k_cache), ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev))
    _lib.check(rc, "tvk_paged_decode_attention")
    if check:
        check_workspace(dev, "decode", "tvk_paged_decode_attention")
    return out


def paged_decode_attention_q8(queries: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                              k_scale: torch.Tensor, v_scale: torch.Tensor, block_tables: torch.Tensor,
                              context_lens: torch.Tensor, n_heads: int, n_kv_heads: int, head_dim: int,
                              block_size: int, max_context_len: Optional[int] = None, *,
                              out: Optional[torch.Tensor] = None, check: bool = False) -> torch.Tensor:
    """``paged_decode_attention`` over a cache held in 8 bits.

    k_cache/v_cache ``torch.float8_e4m3fn`` codes [N,block_size,Hkv,D], k_scale/v_scale
    fp32 [N,Hkv], one scale per block and KV head (``layers.write_kv_slots_q8`` fills
    them; a value is code * scale).  queries [B,1,Hq,D] in fp32, fp16 or bf16;
    everything else, and the masking, as in ``paged_decode_attention``.  Returns
    [B,1,Hq,D] in the dtype of the queries.
    """
    dev = _lib.same_device(queries, k_cache, v_cache, k_scale, v_scale, block_tables, context_lens)
    qs, ks, ts = queries.shape, k_cache.shape, block_tables.shape
    B = qs[0] if qs else 0
    if qs[1:] != (1, n_heads, head_dim):
        raise ValueError(f"queries must be [B,1,{n_heads},{head_dim}], got {tuple(qs)}")
    if ks[1:] != (block_size, n_kv_heads, head_dim) or v_cache.shape != ks:
        raise ValueError(f"k_cache/v_cache must be [N,{block_size},{n_kv_heads},{head_dim}], got "
                         f"{tuple(ks)} / {tuple(v_cache.shape)}")
    if k_cache.dtype != torch.float8_e4m3fn or v_cache.dtype != torch.float8_e4m3fn:
        raise TypeError("k_cache and v_cache must be float8_e4m3fn")
    if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
        raise TypeError("k_scale and v_scale must be float32")
    if k_scale.shape != (ks[0], n_kv_heads) or v_scale.shape != (ks[0], n_kv_heads):
        raise ValueError(f"k_scale/v_scale must be [{ks[0]},{n_kv_heads}], got {tuple(k_scale.shape)} / "
                         f"{tuple(v_scale.shape)}")
    if block_tables.dtype != torch.int32 or context_lens.dtype != torch.int32:
        raise TypeError("block_tables and context_lens must be int32")
    if len(ts) != 2 or ts[0] != B or context_lens.shape != (B,):
        raise ValueError("block_tables must be [B,max_blocks] and context_lens [B]")
    if not (queries.is_contiguous() and k_cache.is_contiguous() and v_cache.is_contiguous()
            and k_scale.is_contiguous() and v_scale.is_contiguous() and block_tables.is_contiguous()
            and context_lens.is_contiguous()):
        raise ValueError("all tensors must be contiguous")
    if out is None:
        out = torch.empty_like(queries)
    elif (out.shape != qs or out.dtype != queries.dtype or out.get_device() != dev or not out.is_contiguous()):
        raise ValueError("out must be a contiguous tensor like queries")
    ws = _workspace_q8(dev, B, n_kv_heads)
    rc = _lib.call_on(
        dev, _lib.lib().tvk_paged_decode_attention_q8, queries.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
        k_scale.data_ptr(), v_scale.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), out.data_ptr(),
        B, n_heads, n_kv_heads, head_dim, block_size, ks[0], ts[1],
        -1 if max_context_len is None else int(max_context_len), _lib.dtype_code(queries), ws.data_ptr(), ws.numel(),
        _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "tvk_paged_decode_attention_q8")
    if check:
        check_workspace(torch.device("cuda", dev), "decode_q8", "tvk_paged_decode_attention_q8")
    return out


def flash_prefill_attention_varlen(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                                   cu_seqlens: torch.Tensor, max_seqlen: int, causal: bool = True, *,
                                   slot_mapping: Optional[torch.Tensor] = None,
                                   k_cache: Optional[torch.Tensor] = None,
                                   v_cache: Optional[torch.Tensor] = None,
                                   out: Optional[torch.Tensor] = None, check: bool = False) -> torch.Tensor:
    """Causal (or full) attention over a ragged batch of prompts packed along tokens.

    q [T,Hq,D], k/v [T,Hkv,D]; ``cu_seqlens`` int32 [n+1] prefix sums of the prompt
    lengths (device); ``max_seqlen`` >= the longest prompt.  With ``slot_mapping``
    (int64 [T], device; -1 skips a token) the kernel also writes each token's k/v
    row into ``k_cache/v_cache`` [N,block_size,Hkv,D] at flat slot
    ``block*block_size + offset`` -- the paged write of llama.py:188-209 fused
    into the attention kernel.  Returns [T,Hq,D].  ``check=True`` synchronises and
    raises ``TvkError`` if a bounded wait inside the kernel timed out.
    """
    tensors = [q, k, v, cu_seqlens] + [t for t in (slot_mapping, k_cache, v_cache) if t is not None]
    dev = _lib.require_cuda(*tensors)
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"q must be [T,Hq,D] and k/v [T,Hkv,D]; got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    if q.dtype != k.dtype or v.dtype != k.dtype:
        raise TypeError("q, k and v must share one dtype")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1:
        raise TypeError("cu_seqlens must be a 1-D int32 tensor")
    for name, t in (("q", q), ("k", k), ("v", v), ("cu_seqlens", cu_seqlens)):
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    n_seqs = cu_seqlens.shape[0] - 1
    num_blocks = block_size = 0
    if slot_mapping is not None:
        if k_cache is None or v_cache is None:
            raise ValueError("slot_mapping needs k_cache and v_cache")
        if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (T,):
            raise TypeError("slot_mapping must be int64 [T]")
        if (k_cache.dim() != 4 or k_cache.shape[2:] != (Hkv, D) or v_cache.shape != k_cache.shape
                or k_cache.dtype != q.dtype or v_cache.dtype != q.dtype
                or not k_cache.is_contiguous() or not v_cache.is_contiguous()):
            raise ValueError("k_cache/v_cache must be contiguous [N,block_size,Hkv,D] in the dtype of q")
        num_blocks, block_size = k_cache.shape[0], k_cache.shape[1]
    if out is None:
        out = torch.empty_like(q)
    L = _lib.lib()
    ws = _workspace(dev, L.tvk_flash_prefill_workspace_size(n_seqs, T), "prefill")
    rc = L.tvk_flash_prefill_attention(
        _lib.ptr(q), _lib.ptr(k), _lib.ptr(v), _lib.ptr(out), _lib.ptr(cu_seqlens), n_seqs, int(max_seqlen), T,
        Hq, Hkv, D, 1 if causal else 0, _lib.dtype_code(q), _lib.ptr(slot_mapping), _lib.ptr(k_cache),
        _lib.ptr(v_cache), num_blocks, block_size, ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev))
    _lib.check(rc, "tvk_flash_prefill_attention")
    if check:
        check_workspace(dev, "prefill", "tvk_flash_prefill_attention")
    return out


def flash_prefill_attention(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                            causal: bool = True) -> torch.Tensor:
    """Flash attention for prefill (tinyvllm/model/llama.py:58-94).

    Inputs [1,L,H,D] (keys/values may have fewer heads, GQA); returns [1,L,Hq,D].
    """
    dev = _lib.require_cuda(queries, keys, values)
    if queries.dim() != 4 or queries.shape[0] != 1:
        raise ValueError("queries must be [1,L,H,D]")
    q = queries[0].contiguous()
    k = keys[0].contiguous()
    v = values[0].contiguous()
    L = q.shape[0]
    cu = torch.tensor([0, L], dtype=torch.int32, device=dev)
    return flash_prefill_attention_varlen(q, k, v, cu, L, causal)[None]
