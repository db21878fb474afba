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


_current = _raw_device if _raw_device is not None else torch.cuda.current_device


def _plain(t, dtype, shape: tuple, dev: int) -> bool:
    """Whether t is a plain contiguous tensor of this type and shape on GPU `dev`
    (a call's usual operand, told in one pass)."""
    return (type(t) is torch.Tensor and t.dtype is dtype and t.shape == shape
            and t.get_device() == dev and t.is_contiguous())


def _rows(t, name: str, n: int, width: int, dtype, dev: int) -> int:
    """Checks rows [n][width] of `dtype` with neighbouring elements; their stride."""
    if _plain(t, dtype, (n, width), dev):
        return width
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.get_device() != dev \
            or t.dtype != dtype:
        raise TypeError(f"{name} must be a {dtype} tensor on cuda:{dev}")
    if t.shape != (n, width):
        raise ValueError(f"{name} must have shape {(n, width)}, got {tuple(t.shape)}")
    s = t.stride()
    if (width > 1 and s[1] != 1) or (n > 1 and s[0] < width):
        raise ValueError(f"{name} must have rows of neighbouring elements that do not overlap")
    return s[0] if n > 1 else max(s[0], width)


def _values(t, name: str, n: int, dtype, dev: int) -> int:
    """Checks n neighbouring values of `dtype`; their address."""
    if not _plain(t, dtype, (n,), dev):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.get_device() != dev \
                or t.dtype != dtype:
            raise TypeError(f"{name} must be a {dtype} tensor on cuda:{dev}")
        raise ValueError(f"{name} must be contiguous with shape {(n,)}, got {tuple(t.shape)}")
    return t.data_ptr()


def _pool(pool, tables, kv_dim: int) -> BatchPool:
    if not isinstance(pool, torch.Tensor) or not pool.is_cuda \
            or pool.dtype not in (torch.float16, torch.int16):
        raise TypeError("pool must be a CUDA float16 (or int16 bits) tensor")
    ps = pool.shape
    if len(ps) != 4 or ps[1] != 2 or ps[3] != kv_dim or not pool.is_contiguous():
        raise ValueError(f"pool must be contiguous [blocks][2][block_size][{kv_dim}], got "
                         f"{tuple(ps)}")
    if not isinstance(tables, torch.Tensor) or not tables.is_cuda \
            or tables.get_device() != pool.get_device() or tables.dtype != torch.int32:
        raise TypeError(f"tables must be an int32 tensor on {pool.device}")
    if tables.dim() != 2:
        raise ValueError("tables must be [requests][blocks]")
    n, blocks = tables.shape
    stride = blocks
    if not tables.is_contiguous():
        s = tables.stride()
        if (blocks > 1 and s[1] != 1) or (n > 1 and s[0] < blocks):
            raise ValueError("tables must be [requests][blocks] with neighbouring entries")
        stride = s[0] if n > 1 else blocks
    return BatchPool(pool.data_ptr(), tables.data_ptr(), ps[0], ps[2], kv_dim, n, blocks, stride)


def _new(shape: tuple, dtype, device, stream, zero: bool = False) -> torch.Tensor:
    """A new tensor that belongs to the call's stream: filled there, and its
    memory free for other uses only behind the call."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return _new(shape, dtype, device, None, zero)
    return (torch.zeros if zero else torch.empty)(shape, dtype=dtype, device=device)


def _workspace(given: Optional[torch.Tensor], need: int, device, stream):
    """(pointer, bytes, tensor) of the caller's workspace or of a new one."""
    if given is None:
        if need == 0:
            return None, 0, None
        given = _new((need,), torch.uint8, device, stream)
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
    kvd, dt = nkv * dph, k.dtype
    d = _pool(pool, tables, kvd)
    dev, T = pool.get_device(), seq.shape[0]
    dtype = _DTYPES.get(dt)
    if dtype is None:
        raise TypeError(f"k must be float32, float16 or bfloat16, got {dt}")
    if dev != _current():
        with torch.cuda.device(dev):
            return batch_append(pool, tables, seq, pos, k, v, nh, nkv, dph, theta, scaling_type,
                                scaling_factor, rotate, q, q_out, k_out, stream)
    sp = _values(seq, "seq", T, torch.int32, dev)
    pp = _values(pos, "pos", T, torch.int32, dev)
    ks = _rows(k, "k", T, kvd, dt, dev)
    vs = _rows(v, "v", T, kvd, dt, dev)
    qp = qop = kop = None
    qs = qos = kos = 0
    if q is not None:
        qs = _rows(q, "q", T, nh * dph, dt, dev)
        if q_out is None:
            q_out = _new((T, nh * dph), dt, pool.device, stream, zero=True)
        qos = _rows(q_out, "q_out", T, nh * dph, dt, dev)
        qp, qop = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out needs q")
    if k_out is not None:
        kos = _rows(k_out, "k_out", T, kvd, dt, dev)
        kop = k_out.data_ptr()
    rope = ctypes.byref(RopeConfig(theta, scaling_type, scaling_factor)) if rotate else None
    check(_native.load().sde_batch_append(
        ctypes.byref(d), sp, pp, T, dtype, k.data_ptr(), ks, v.data_ptr(), vs, kop, kos, qp, qs,
        qop, qos, nh, nkv, dph, rope, _stream(stream)), "batch_append")
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
    dev, n, dt, width = pool.get_device(), d.n_seqs, q.dtype, nh * dph
    dtype = _DTYPES.get(dt)
    if dtype is None:
        raise TypeError(f"q must be float32, float16 or bfloat16, got {dt}")
    if dev != _current():
        with torch.cuda.device(dev):
            return batch_attention(q, pool, tables, lens, nh, nkv, dph, n_queries, max_len, out,
                                   workspace, stream)
    lp = _values(lens, "lens", n, torch.int32, dev)
    qs = _rows(q, "q", n * n_queries, width, dt, dev)
    if max_len is None:
        max_len = d.max_blocks * d.block_size
    if out is None:
        out, os = _new((n * n_queries, width), dt, pool.device, stream), width
    else:
        os = _rows(out, "out", n * n_queries, width, dt, dev)
    lib = _native.load()
    ptr, size, workspace = _workspace(
        workspace, lib.sde_batch_attention_workspace_size(n, nh, nkv, dph, n_queries, max_len,
                                                          d.block_size), pool.device, stream)
    check(lib.sde_batch_attention(ctypes.byref(d), lp, n_queries, max_len, dtype, q.data_ptr(), qs,
                                  out.data_ptr(), os, nh, nkv, dph, ptr, size, _stream(stream)),
          "batch_attention")
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
    dt, dev, T = q.dtype, q.get_device(), q.shape[0]
    if dev != _current():
        with torch.cuda.device(dev):
            return prompt_attention(q, k, v, starts, nh, nkv, dph, out, stream)
    qs = _rows(q, "q", T, nh * dph, dt, dev)
    ks = _rows(k, "k", T, nkv * dph, dt, dev)
    vs = _rows(v, "v", T, nkv * dph, dt, dev)
    if not isinstance(starts, torch.Tensor) or starts.dim() != 1 or starts.shape[0] < 1:
        raise ValueError("starts must have one entry per sequence and one for the end")
    n = starts.shape[0]
    sp = _values(starts, "starts", n, torch.int32, dev)
    if out is None:
        out, os = _new((T, nh * dph), dt, q.device, stream, zero=True), nh * dph
    else:
        os = _rows(out, "out", T, nh * dph, dt, dev)
    check(_native.load().sde_prompt_attention(
        sp, n - 1, T, dtype, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, out.data_ptr(),
        os, nh, nkv, dph, _stream(stream)), "prompt_attention")
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
    dev, (n, V) = logits.get_device(), logits.shape
    if dev != _current():
        with torch.cuda.device(dev):
            return sample(logits, u, temperature, top_k, top_p, min_p, tokens, probs, workspace,
                          stream)
    f32, i32 = torch.float32, torch.int32
    stride = _rows(logits, "logits", n, V, logits.dtype, dev)
    up = _values(u, "u", n, f32, dev)
    tp = None if temperature is None else _values(temperature, "temperature", n, f32, dev)
    kp = None if top_k is None else _values(top_k, "top_k", n, i32, dev)
    pp = None if top_p is None else _values(top_p, "top_p", n, f32, dev)
    mp = None if min_p is None else _values(min_p, "min_p", n, f32, dev)
    if tokens is None:
        tokens = _new((n,), i32, logits.device, stream)
    if probs is None:
        probs = _new((n,), f32, logits.device, stream)
    lib = _native.load()
    ptr, size, workspace = _workspace(workspace, lib.sde_sample_workspace_size(n, V),
                                      logits.device, stream)
    check(lib.sde_sample(
        logits.data_ptr(), stride, dtype, n, V, up, tp, kp, pp, mp,
        _values(tokens, "tokens", n, i32, dev), _values(probs, "probs", n, f32, dev), ptr, size,
        _stream(stream)), "sample")
    return tokens, probs
