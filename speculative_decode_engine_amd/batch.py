"""Steps over several requests that share one paged pool: a ctypes mirror of
sde_batch_append, sde_batch_attention, sde_prompt_attention and sde_sample
(include/sde_paged_kv.h).

The pool has KVCache's layout, float16 (or its int16 bits)
[blocks][2][block_size][kv_dim]; `KVCache.pool_blocks_view()` is one.  A step of
a batch is, per layer,

    batch_append(pool, tables, seq, pos, k, v, nh, nkv, dph, q=q, q_out=q)
    out = batch_attention(q, pool, tables, lens, nh, nkv, dph)

(new prompts, packed, take `prompt_attention` over the rotated rows) and at its
end, over the rows of logits,

    tokens, probs = sample(logits, u, temperature, top_k, top_p, min_p)

with `tables` the layer's block tables, one row per request, and positions and
lengths on the device: a captured graph replays with new ones.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _native
from ._native import BatchPool, RopeConfig, check
from .kv_cache import _raw_device, _stream

_DTYPES = {torch.float32: _native.SDE_F32, torch.float16: _native.SDE_F16,
           torch.bfloat16: _native.SDE_BF16}


class _On:
    """The buffers' device made current for a call where it is not already
    (streams and launches belong to the current device)."""

    def __init__(self, device):
        self.guard = None
        if device.index != (_raw_device() if _raw_device else torch.cuda.current_device()):
            self.guard = torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _rows(t, name: str, n: int, width: int, dtype, device) -> int:
    """Checks rows [n][width] of `dtype` with neighbouring elements; their stride."""
    if not isinstance(t, torch.Tensor) or t.device != device or t.dtype != dtype:
        raise TypeError(f"{name} must be a {dtype} tensor on {device}")
    if t.shape != (n, width):
        raise ValueError(f"{name} must have shape {(n, width)}, got {tuple(t.shape)}")
    s = t.stride()
    if (width > 1 and s[1] != 1) or (n > 1 and s[0] < width):
        raise ValueError(f"{name} must have rows of neighbouring elements that do not overlap")
    return s[0] if n > 1 else max(s[0], width)


def _ints(t, name: str, n: int, device) -> None:
    if not isinstance(t, torch.Tensor) or t.device != device or t.dtype != torch.int32:
        raise TypeError(f"{name} must be an int32 tensor on {device}")
    if t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous with shape {(n,)}, got {tuple(t.shape)}")


def _pool(pool, tables, kv_dim: int) -> BatchPool:
    if not isinstance(pool, torch.Tensor) or pool.device.type != "cuda" \
            or pool.dtype not in (torch.float16, torch.int16):
        raise TypeError("pool must be a CUDA float16 (or int16 bits) tensor")
    if pool.dim() != 4 or pool.shape[1] != 2 or pool.shape[3] != kv_dim \
            or not pool.is_contiguous():
        raise ValueError(f"pool must be contiguous [blocks][2][block_size][{kv_dim}], got "
                         f"{tuple(pool.shape)}")
    if not isinstance(tables, torch.Tensor) or tables.device != pool.device \
            or tables.dtype != torch.int32:
        raise TypeError(f"tables must be an int32 tensor on {pool.device}")
    if tables.dim() != 2 or (tables.shape[1] > 1 and tables.stride(1) != 1) \
            or (tables.shape[0] > 1 and tables.stride(0) < tables.shape[1]):
        raise ValueError("tables must be [requests][blocks] with neighbouring entries")
    n, blocks = tables.shape
    return BatchPool(pool.data_ptr(), tables.data_ptr(), pool.shape[0], pool.shape[2], kv_dim, n,
                     blocks, tables.stride(0) if n > 1 else blocks)


def _workspace(given: Optional[torch.Tensor], need: int, device, stream):
    """(pointer, bytes, tensor) of the caller's workspace or of a new one."""
    if given is None:
        if need == 0:
            return None, 0, None
        given = torch.empty(need, dtype=torch.uint8, device=device)
        if stream is not None:
            given.record_stream(stream)
        return given.data_ptr(), need, given
    if given.device != device or not given.is_contiguous():
        raise ValueError(f"workspace must be a contiguous tensor on {device}")
    return given.data_ptr(), given.numel() * given.element_size(), given


def batch_append(pool: torch.Tensor, tables: torch.Tensor, seq: torch.Tensor, pos: torch.Tensor,
                 k: torch.Tensor, v: torch.Tensor, nh: int, nkv: int, dph: int,
                 theta: float = 10000.0, scaling_type: int = 0, scaling_factor: float = 1.0,
                 rotate: bool = True, q: Optional[torch.Tensor] = None,
                 q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None,
                 stream=None) -> Optional[torch.Tensor]:
    """Rotates and appends tokens of several requests in one launch: token t
    belongs to request seq[t] (below 0: padding, left out) at position pos[t]
    (int32).  k and v, rows [T][nkv*dph] of float32, float16 or bfloat16, go to
    the pool as fp16, k rotated by rotate-half RoPE (rotate=False: as it is).
    With q, [T][nh*dph] of the same type, its rotation goes to q_out (allocated
    when None; q itself: in place) and is returned; k_out takes the rotated k as
    well.  Rows may be slices of a fused projection."""
    d = _pool(pool, tables, nkv * dph)
    dev, T = pool.device, seq.shape[0]
    dtype = _DTYPES.get(k.dtype)
    if dtype is None:
        raise TypeError(f"k must be float32, float16 or bfloat16, got {k.dtype}")
    _ints(seq, "seq", T, dev)
    _ints(pos, "pos", T, dev)
    ks = _rows(k, "k", T, nkv * dph, k.dtype, dev)
    vs = _rows(v, "v", T, nkv * dph, k.dtype, dev)
    qs = qos = kos = 0
    if q is not None:
        qs = _rows(q, "q", T, nh * dph, k.dtype, dev)
        if q_out is None:
            q_out = torch.zeros(T, nh * dph, dtype=q.dtype, device=dev)
        qos = _rows(q_out, "q_out", T, nh * dph, k.dtype, dev)
    elif q_out is not None:
        raise ValueError("q_out needs q")
    if k_out is not None:
        kos = _rows(k_out, "k_out", T, nkv * dph, k.dtype, dev)
    rope = ctypes.byref(RopeConfig(theta, scaling_type, scaling_factor)) if rotate else None
    with _On(dev):
        check(_native.load().sde_batch_append(
            ctypes.byref(d), seq.data_ptr(), pos.data_ptr(), T, dtype, k.data_ptr(), ks,
            v.data_ptr(), vs, None if k_out is None else k_out.data_ptr(), kos,
            None if q is None else q.data_ptr(), qs, None if q is None else q_out.data_ptr(), qos,
            nh, nkv, dph, rope, _stream(stream)), "batch_append")
    return q_out


def batch_attention_workspace_size(n_seqs: int, nh: int, nkv: int, dph: int, n_queries: int,
                                   max_len: int, block_size: int) -> int:
    return int(_native.load().sde_batch_attention_workspace_size(
        n_seqs, nh, nkv, dph, n_queries, max_len, block_size))


def batch_attention(q: torch.Tensor, pool: torch.Tensor, tables: torch.Tensor,
                    lens: torch.Tensor, nh: int, nkv: int, dph: int, n_queries: int = 1,
                    max_len: Optional[int] = None, out: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Causal attention of each request's newest n_queries tokens over its own
    positions: q [n_seqs*n_queries][nh*dph] (float32, float16 or bfloat16), lens
    int32 [n_seqs] the lengths with the new tokens; query i of request s sees
    positions [0, lens[s] - n_queries + i], and one that sees nothing gives
    zeros.  max_len bounds the lengths (default: what the tables hold); the
    launch is planned for it, so a tight bound is faster.  The workspace
    (batch_attention_workspace_size bytes) is taken from torch's allocator when
    None."""
    d = _pool(pool, tables, nkv * dph)
    dev, n = pool.device, tables.shape[0]
    dtype = _DTYPES.get(q.dtype)
    if dtype is None:
        raise TypeError(f"q must be float32, float16 or bfloat16, got {q.dtype}")
    _ints(lens, "lens", n, dev)
    qs = _rows(q, "q", n * n_queries, nh * dph, q.dtype, dev)
    if max_len is None:
        max_len = d.max_blocks * d.block_size
    with _On(dev):
        if out is None:
            out = torch.empty(n * n_queries, nh * dph, dtype=q.dtype, device=dev)
        os = _rows(out, "out", n * n_queries, nh * dph, q.dtype, dev)
        lib = _native.load()
        ptr, size, workspace = _workspace(
            workspace, lib.sde_batch_attention_workspace_size(n, nh, nkv, dph, n_queries, max_len,
                                                              d.block_size), dev, stream)
        check(lib.sde_batch_attention(
            ctypes.byref(d), lens.data_ptr(), n_queries, max_len, dtype, q.data_ptr(), qs,
            out.data_ptr(), os, nh, nkv, dph, ptr, size, _stream(stream)), "batch_attention")
    return out


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor,
                     nh: int, nkv: int, dph: int, out: Optional[torch.Tensor] = None,
                     stream=None) -> torch.Tensor:
    """Causal attention of packed prompts within themselves: sequence b's tokens
    are rows starts[b] .. starts[b+1]-1 (int32, on the device) of q and out
    [T][nh*dph] and of k and v [T][nkv*dph], float16 or bfloat16, rotated
    already.  Rows may be slices of a fused projection (multiples of 16 bytes).
    Rows outside the sequences are left as they were (zeros where out is
    allocated here)."""
    if not isinstance(q, torch.Tensor) or q.device.type != "cuda" or q.dim() != 2:
        raise TypeError("q must be a 2-D CUDA tensor")
    dtype = _DTYPES.get(q.dtype)
    if dtype is None or dtype == _native.SDE_F32:
        raise TypeError(f"q must be float16 or bfloat16, got {q.dtype}")
    dev, T = q.device, q.shape[0]
    qs = _rows(q, "q", T, nh * dph, q.dtype, dev)
    ks = _rows(k, "k", T, nkv * dph, q.dtype, dev)
    vs = _rows(v, "v", T, nkv * dph, q.dtype, dev)
    if not isinstance(starts, torch.Tensor) or starts.dim() != 1 or starts.shape[0] < 1:
        raise ValueError("starts must have one entry per sequence and one for the end")
    _ints(starts, "starts", starts.shape[0], dev)
    with _On(dev):
        if out is None:
            out = torch.zeros(T, nh * dph, dtype=q.dtype, device=dev)
        os = _rows(out, "out", T, nh * dph, q.dtype, dev)
        check(_native.load().sde_prompt_attention(
            starts.data_ptr(), starts.shape[0] - 1, T, dtype, q.data_ptr(), qs, k.data_ptr(), ks,
            v.data_ptr(), vs, out.data_ptr(), os, nh, nkv, dph, _stream(stream)),
            "prompt_attention")
    return out


def sample_workspace_size(n_rows: int, vocab: int) -> int:
    return int(_native.load().sde_sample_workspace_size(n_rows, vocab))


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Optional[torch.Tensor] = None,
           top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
           min_p: Optional[torch.Tensor] = None, tokens: Optional[torch.Tensor] = None,
           probs: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
           stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """One token per row of logits [rows][vocab] (float32, float16 or bfloat16),
    drawn with the random numbers u (float32 [rows], in [0, 1)): weights
    exp(x / temperature), the top_k largest, of those the shortest run that
    reaches top_p of their weight, of those the ones of at least min_p times the
    largest; the token where the kept weight, summed by index, passes u of it.
    Parameters are float32 (top_k int32) tensors of one value per row, or None
    (temperature 1, no filter); a temperature below 1e-6 takes the largest
    logit.  Returns tokens int32 [rows] (-1 where every logit is -inf or NaN)
    and each one's probability among those kept.  The workspace
    (sample_workspace_size bytes) is taken from torch's allocator when None."""
    if not isinstance(logits, torch.Tensor) or logits.device.type != "cuda" or logits.dim() != 2:
        raise TypeError("logits must be a 2-D CUDA tensor")
    dtype = _DTYPES.get(logits.dtype)
    if dtype is None:
        raise TypeError(f"logits must be float32, float16 or bfloat16, got {logits.dtype}")
    dev, (n, V) = logits.device, logits.shape
    stride = _rows(logits, "logits", n, V, logits.dtype, dev)
    for t, name, want in ((u, "u", torch.float32), (temperature, "temperature", torch.float32),
                          (top_k, "top_k", torch.int32), (top_p, "top_p", torch.float32),
                          (min_p, "min_p", torch.float32), (tokens, "tokens", torch.int32),
                          (probs, "probs", torch.float32)):
        if t is None and name != "u":
            continue
        if not isinstance(t, torch.Tensor) or t.device != dev or t.dtype != want:
            raise TypeError(f"{name} must be a {want} tensor on {dev}")
        if t.shape != (n,) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous with shape {(n,)}, got {tuple(t.shape)}")
    with _On(dev):
        if tokens is None:
            tokens = torch.empty(n, dtype=torch.int32, device=dev)
        if probs is None:
            probs = torch.empty(n, dtype=torch.float32, device=dev)
        lib = _native.load()
        ptr, size, workspace = _workspace(workspace, lib.sde_sample_workspace_size(n, V), dev,
                                          stream)
        check(lib.sde_sample(
            logits.data_ptr(), stride, dtype, n, V, u.data_ptr(),
            None if temperature is None else temperature.data_ptr(),
            None if top_k is None else top_k.data_ptr(),
            None if top_p is None else top_p.data_ptr(),
            None if min_p is None else min_p.data_ptr(), tokens.data_ptr(), probs.data_ptr(),
            ptr, size, _stream(stream)), "sample")
    return tokens, probs
