"""Serving: attention over a key/value cache held in 4 bits.

The rest of the framework attends the tokens of one call to each other. A server that generates text
attends each step's new tokens to everything before them. This module keeps those keys and values in
4.25 bits per element, in blocks that requests of unequal length take from one pool:

    cache = kv4.allocate(num_blocks, heads_kv, head_dim)            # one per layer
    step = kv4.plan(lens, new, table, free, used, block_size=cache.block_size, tokens=T)
    kv4.write(cache, k, v, step.slots)                              # the step's keys and values, stored
    o = kv4.attention(q, cache, table, step.lens, step.cu)          # its queries over all of the cache

``plan`` runs once per step, on the GPU, from the requests' lengths there; ``write`` and ``attention`` once per
layer. q: (B, Hq, N, D), k and v: (B, Hkv, N, D), fp16 or bf16, D in {64, 128, 256, 512}, strided views
read in place, as everywhere in the framework. A call's tokens are counted through its rows, token t being
row t % N of batch entry t // N: a packed step is (1, H, T, D), a step of one token per request may be
(B, H, 1, D).

Format (MXFP4): 32 neighbouring channels of a token and head share a power of two; an element is a sign
and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6. The largest of the 32 lands in (3.5, 7] times the power of two, and
values round to the nearest (ties to the even code, above 6 to 6): an error of 11% (rms) on normally
distributed values. Infinities and NaN are kept as NaN: a query that attends to such a token answers NaN,
no other does.

Every call launches on its tensors' device and that device's current stream, reads no device value on the
host, and can be captured into a graph. There is no CPU path: unsupported inputs raise before anything is
launched.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib
from .attention import _DTYPES, _check_softcap, _default_scale, _needs_copy, _stream
from .registry import lookup

BLOCK_SIZES = (32, 64, 128, 256, 512, 1024)


class Cache:
    """A layer's cache: ``codes`` (num_blocks, Hkv, 2, block_size, D / 2) and ``scales`` (num_blocks, Hkv, 2,
    block_size, D / 32), uint8, contiguous, on one GPU, for rows of ``dtype``. Blocks need no initial
    contents. The bytes inside a block are in the order the kernels read (csrc/gfa_kv4.h)."""

    __slots__ = ("codes", "scales", "dtype", "num_blocks", "heads_kv", "block_size", "head_dim")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype):
        if dtype not in _DTYPES:
            raise TypeError(f"dtype {dtype} not supported (fp16 / bf16)")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("codes and scales must be uint8")
        if codes.dim() != 5 or scales.dim() != 5:
            raise ValueError("codes and scales must be 5-D (num_blocks, heads_kv, 2, block_size, bytes)")
        n, h, two, bs, half = codes.shape
        lookup(2 * half)
        if two != 2 or tuple(scales.shape) != (n, h, 2, bs, half // 16):
            raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not belong together")
        if bs not in BLOCK_SIZES:
            raise ValueError(f"block_size={bs} not supported; options {BLOCK_SIZES}")
        if n == 0 or h == 0:
            raise ValueError("a cache needs blocks and heads")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("codes and scales must be contiguous")
        if not (codes.is_cuda and scales.is_cuda) or codes.device != scales.device:
            raise ValueError("codes and scales must be on one GPU (the engine has no CPU path)")
        self.codes, self.scales, self.dtype = codes, scales, dtype
        self.num_blocks, self.heads_kv, self.block_size, self.head_dim = n, h, bs, 2 * half

    def __repr__(self) -> str:
        return (f"kv4.Cache(num_blocks={self.num_blocks}, heads_kv={self.heads_kv}, head_dim={self.head_dim}, "
                f"block_size={self.block_size}, dtype={self.dtype}, device={self.codes.device})")


def allocate(num_blocks: int, heads_kv: int, head_dim: int, block_size: int = 64, dtype: torch.dtype = torch.bfloat16,
             device="cuda") -> Cache:
    """A new cache of ``num_blocks`` blocks of ``block_size`` tokens: 1.0625 bytes per token, KV head and channel."""
    lookup(head_dim)
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size={block_size} not supported; options {BLOCK_SIZES}")
    shape = (int(num_blocks), int(heads_kv), 2, block_size)
    return Cache(torch.empty((*shape, head_dim // 2), dtype=torch.uint8, device=device),
                 torch.empty((*shape, head_dim // 32), dtype=torch.uint8, device=device), dtype)


class Plan(NamedTuple):
    """A step's plan (``plan``)."""

    slots: torch.Tensor      # (tokens,) int64: where each new token is stored; -1: nowhere
    positions: torch.Tensor  # (tokens,) int32: its position in its request
    cu: torch.Tensor         # (requests + 1,) int32: the requests' first tokens
    lens: torch.Tensor       # (requests,) int32: tokens with the new ones
    used: torch.Tensor       # (1,) int32: entries of the free list handed out


def _gpu(name: str, t: torch.Tensor, device, dtype, shape) -> torch.Tensor:
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != len(shape) or any(a != b for a, b in zip(t.shape, shape) if b is not None):
        want = tuple("*" if x is None else x for x in shape)
        raise ValueError(f"{name} must have shape {want}, got {tuple(t.shape)}")
    if t.device != device or not t.is_cuda:
        raise ValueError(f"{name} must be on the call's GPU ({device}), is on {t.device}")
    return t


def _table(table: torch.Tensor, device, requests) -> int:
    _gpu("table", table, device, torch.int32, (requests, None))
    if table.shape[0] == 0 or table.shape[1] == 0:
        raise ValueError("empty block table")
    if table.stride(1) != 1 or (table.shape[0] > 1 and table.stride(0) < table.shape[1]):
        raise ValueError("table rows must be contiguous and apart from each other")
    return table.stride(0) if table.shape[0] > 1 else table.shape[1]


def plan(lens: torch.Tensor, new: torch.Tensor, table: torch.Tensor, free: torch.Tensor, used: torch.Tensor, *,
         block_size: int, tokens: int) -> Plan:
    """Places for a step's new tokens, in one launch.

    lens, new: (B,) int32, tokens each request holds and gets (0 for a request without new ones). table: (B, M) int32,
    its blocks by position, filled in place for the blocks the request grows by. free: (F,) int32 ids of
    free blocks, of which the first ``used`` ((1,) int32) are handed out; requests take the next ones in their
    order. ``tokens``: the step's static token count, at least the sum of ``new``; what lies behind is padding
    (slot -1). A table entry past the free list is -1, and so are the slots there; ``Plan.used`` above F tells
    of it. The next step takes ``Plan.lens`` and ``Plan.used``."""
    dev = lens.device
    _gpu("lens", lens, dev, torch.int32, (None,))
    B = lens.shape[0]
    _gpu("new", new, dev, torch.int32, (B,))
    stride = _table(table, dev, B)
    _gpu("free", free, dev, torch.int32, (None,))
    _gpu("used", used, dev, torch.int32, (1,))
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size={block_size} not supported; options {BLOCK_SIZES}")
    tokens = int(tokens)
    if tokens < 0 or tokens >= 1 << 31:
        raise ValueError(f"tokens={tokens} must be in [0, 2^31)")
    lens, new, free = lens.contiguous(), new.contiguous(), free.contiguous()
    out = Plan(torch.empty((tokens,), dtype=torch.int64, device=dev), torch.empty((tokens,), dtype=torch.int32, device=dev),
               torch.empty((B + 1,), dtype=torch.int32, device=dev), torch.empty((B,), dtype=torch.int32, device=dev),
               torch.empty((1,), dtype=torch.int32, device=dev))
    a = _lib.Kv4PlanArgs()
    a.lens, a.fresh, a.table, a.table_stride = lens.data_ptr(), new.data_ptr(), table.data_ptr(), stride
    a.free_ids, a.used = free.data_ptr(), used.data_ptr()
    a.requests, a.table_width, a.free_count, a.block_size, a.tokens = B, table.shape[1], free.shape[0], block_size, tokens
    a.slots, a.positions, a.cu, a.lens_out, a.used_out = (t.data_ptr() for t in out)
    a.stream = _stream(dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().gfa_kv4_plan(ctypes.byref(a)))
    return out


def _cache_args(cache: Cache) -> _lib.Kv4Cache:
    return _lib.Kv4Cache(cache.codes.data_ptr(), cache.scales.data_ptr(), cache.num_blocks, cache.heads_kv,
                         cache.block_size, cache.head_dim, _DTYPES[cache.dtype])


def _check_rows(name: str, t: torch.Tensor, cache: Cache, heads: Optional[int]) -> None:
    if t.dim() != 4:
        raise ValueError(f"{name} must be 4-D (B, H, N, D)")
    if t.dtype != cache.dtype:
        raise TypeError(f"{name} is {t.dtype}, the cache is for {cache.dtype}")
    if t.shape[3] != cache.head_dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} {tuple(t.shape)} does not fit a cache of {cache.heads_kv} heads of dim {cache.head_dim}")
    if t.device != cache.codes.device:
        raise ValueError(f"{name} must be on the cache's GPU ({cache.codes.device}), is on {t.device}")


def _rows_call(fn: str, cache: Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    a = _lib.Kv4RowsArgs()
    a.cache = _cache_args(cache)
    a.k, a.v, a.k_strides, a.v_strides = k.data_ptr(), v.data_ptr(), _lib.strides_of(k), _lib.strides_of(v)
    a.batch, a.seq_len, a.slots = k.shape[0], k.shape[2], slots.data_ptr()
    a.stream = _stream(k.device)
    with torch.cuda.device(k.device):
        _lib.check(getattr(_lib.load(), fn)(ctypes.byref(a)))


def write(cache: Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Store k, v (B, Hkv, N, D) in the cache, token t at ``slots[t]`` (int64, B N of them). A slot outside the
    cache (-1) stores nothing; the slots of one call must differ."""
    _check_rows("k", k, cache, cache.heads_kv)
    _check_rows("v", v, cache, cache.heads_kv)
    if k.shape != v.shape:
        raise ValueError(f"shape mismatch: k {tuple(k.shape)}, v {tuple(v.shape)}")
    _gpu("slots", slots, k.device, torch.int64, (k.shape[0] * k.shape[2],))
    if slots.shape[0] == 0:
        return
    k, v = (t.contiguous() if _needs_copy(t) else t for t in (k, v))
    _rows_call("gfa_kv4_write", cache, k, v, slots.contiguous())


def read(cache: Cache, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values at ``slots`` (int64, (T,)), as (1, Hkv, T, D) of the cache's dtype; zeros for a slot
    outside the cache."""
    _gpu("slots", slots, cache.codes.device, torch.int64, (None,))
    shape = (slots.shape[0], cache.heads_kv, cache.head_dim)
    k, v = (torch.empty(shape, dtype=cache.dtype, device=slots.device)[None].transpose(1, 2) for _ in range(2))
    if slots.shape[0]:
        _rows_call("gfa_kv4_read", cache, k, v, slots.contiguous())
    return k, v


def attention(q: torch.Tensor, cache: Cache, table: torch.Tensor, lens: torch.Tensor, cu: Optional[torch.Tensor] = None, *,
              max_new: Optional[int] = None, causal: bool = True, slide_size: int = 0, scale: Optional[float] = None,
              softcap: Optional[float] = None) -> torch.Tensor:
    """Attention of a step's new tokens over the cache, which holds their own keys and values already.

    q: (B, Hq, N, D), Hq a multiple of the cache's heads. table: (R, M) int32, lens: (R,) int32 tokens of each
    request with its new ones (``Plan.lens``), cu: (R + 1,) int32 the requests' first tokens in q (``Plan.cu``);
    without it every request has B N / R tokens. A request's new tokens are its last ones: the one at
    position p attends to positions <= p, with ``slide_size`` W > 0 only to those > p - W, without ``causal``
    (cross attention) to all of them. Positions whose table entry is no block are not attended to. A row that
    attends to nothing is 0, and so are rows behind the last request's tokens.

    ``max_new``: the most new tokens of any request, if known (1 for a decoding step): it only chooses
    kernels. ``scale`` defaults to 1/sqrt(D); ``softcap`` as in ``flash_attn_gqa_train``. There is no gradient."""
    _check_rows("q", q, cache, None)
    B, Hq, N, D = q.shape
    if Hq == 0 or Hq % cache.heads_kv != 0:
        raise ValueError(f"N_Q_HEADS={Hq} must be a multiple of N_KV_HEADS={cache.heads_kv}")
    if B == 0 or N == 0:
        raise ValueError("empty sequence or batch")
    if torch.is_grad_enabled() and q.requires_grad:
        raise NotImplementedError("attention over the cache has no gradient (call it under torch.no_grad())")
    dev = q.device
    _gpu("lens", lens, dev, torch.int32, (None,))
    R = lens.shape[0]
    stride = _table(table, dev, R)
    if cu is not None:
        cu = _gpu("cu", cu, dev, torch.int32, (R + 1,)).contiguous()
    elif B * N % R:
        raise ValueError(f"{B * N} tokens do not divide among {R} requests (pass cu)")
    slide_size = int(slide_size or 0)
    if slide_size < 0:
        raise ValueError("slide_size must be >= 0")
    if max_new is not None and int(max_new) < 1:
        raise ValueError("max_new must be at least 1")
    cap = _check_softcap(softcap)
    if _needs_copy(q):
        q = q.contiguous()
    o = torch.empty_like(q)
    if _needs_copy(o):
        o = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lens = lens.contiguous()
    a = _lib.Kv4AttnArgs()
    a.cache = _cache_args(cache)
    a.q, a.o, a.q_strides, a.o_strides = q.data_ptr(), o.data_ptr(), _lib.strides_of(q), _lib.strides_of(o)
    a.batch, a.heads_q, a.seq_len, a.requests = B, Hq, N, R
    a.table, a.table_stride, a.lens = table.data_ptr(), stride, lens.data_ptr()
    a.cu = cu.data_ptr() if cu is not None else None
    a.table_width, a.causal, a.window = table.shape[1], int(bool(causal)), min(slide_size, (1 << 31) - 1)
    a.max_new = min(int(max_new), (1 << 31) - 1) if max_new is not None else 0
    a.scale, a.softcap = _default_scale(D, scale), cap
    a.stream = _stream(dev)
    lib = _lib.load()
    need = int(lib.gfa_kv4_attn_workspace_bytes(ctypes.byref(a)))
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    a.workspace, a.workspace_bytes = (ws.data_ptr() if need else None), need
    with torch.cuda.device(dev):
        _lib.check(lib.gfa_kv4_attn(ctypes.byref(a)))
    return o
