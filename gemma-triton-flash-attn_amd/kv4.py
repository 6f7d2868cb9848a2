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

from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .attention import _DTYPES, _ORDINARY, _check_softcap, _default_scale
from .ops import _out_like
from .registry import lookup

BLOCK_SIZES = (32, 64, 128, 256, 512, 1024)


class Cache:
    """A layer's cache: ``codes`` (num_blocks, Hkv, 2, block_size, D / 2) and ``scales`` (num_blocks, Hkv, 2,
    block_size, D / 32), uint8, contiguous, on one GPU, for rows of ``dtype``. Blocks need no initial
    contents. The bytes inside a block are in the order the kernels read (csrc/gfa_kv4.h)."""

    __slots__ = ("codes", "scales", "dtype")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype):
        if dtype not in _DTYPES:
            raise TypeError(f"dtype {dtype} not supported (fp16 / bf16)")
        if _plain(codes):
            _lib.native().kv4_cache(codes, scales)
        self.codes, self.scales, self.dtype = codes, scales, dtype

    num_blocks = property(lambda self: self.codes.shape[0])
    heads_kv = property(lambda self: self.codes.shape[1])
    block_size = property(lambda self: self.codes.shape[3])
    head_dim = property(lambda self: 2 * self.codes.shape[4])

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


def _plain(t: torch.Tensor) -> bool:
    """Whether a call goes straight to the C++ host path: ordinary tensors outside traces, transforms and modes, which
    see the registered ops instead (the same path behind them)."""
    return type(t) in _ORDINARY and _lib.plain_setting()


def _refuse_gradients(what: str, a: torch.Tensor, b: torch.Tensor) -> None:
    if (a.requires_grad or b.requires_grad) and torch.is_grad_enabled():
        raise NotImplementedError(f"{what} has no gradient (call it under torch.no_grad())")
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in (a, b)):
        raise NotImplementedError(f"{what} has no gradient, in forward mode neither")


def plan(lens: torch.Tensor, new: torch.Tensor, table: torch.Tensor, free: torch.Tensor, used: torch.Tensor, *,
         block_size: int, tokens: int) -> Plan:
    """Places for a step's new tokens, in one launch.

    lens, new: (B,) int32, tokens each request holds and gets (0 for a request without new ones). table: (B, M) int32,
    its blocks by position, filled in place for the blocks the request grows by. free: (F,) int32 ids of
    free blocks, of which the first ``used`` ((1,) int32) are handed out; requests take the next ones in their
    order. ``tokens``: the step's static token count, at least the sum of ``new``; what lies behind is padding
    (slot -1). A table entry past the free list is -1, and so are the slots there; ``Plan.used`` above F tells
    of it. A request that outgrows the table's M blocks takes them from the free list all the same: they stand in no
    table, and the slots there are -1. The next step takes ``Plan.lens`` and ``Plan.used`` (outside of torch.compile views
    of one allocation with ``positions`` and ``cu``)."""
    if _plain(lens):
        return Plan(*_lib.native().kv4_plan(lens, new, table, free, used, block_size, tokens, False))
    return Plan(*torch.ops.gfa.kv4_plan(lens, new, table, free, used, block_size, tokens))


def write(cache: Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Store k, v (B, Hkv, N, D) in the cache, token t at ``slots[t]`` (int64, B N of them). A slot outside the
    cache (-1) stores nothing; the slots of one call must differ. There is no gradient."""
    _refuse_gradients("a write to the cache", k, v)
    fn = _lib.native().kv4_write if _plain(k) else torch.ops.gfa.kv4_write
    fn(cache.codes, cache.scales, cache.dtype is torch.bfloat16, k, v, slots)


def read(cache: Cache, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values at ``slots`` (int64, (T,)), as (1, Hkv, T, D) of the cache's dtype; zeros for a slot
    outside the cache. Outside of torch.compile both are views of one allocation: whoever keeps one keeps both."""
    if _plain(slots):
        return _lib.native().kv4_read(cache.codes, cache.scales, cache.dtype is torch.bfloat16, slots, False)
    return torch.ops.gfa.kv4_read(cache.codes, cache.scales, cache.dtype is torch.bfloat16, slots)


def attention(q: torch.Tensor, cache: Cache, table: torch.Tensor, lens: torch.Tensor, cu: Optional[torch.Tensor] = None, *,
              max_new: Optional[int] = None, causal: bool = True, slide_size: int = 0, scale: Optional[float] = None,
              softcap: Optional[float] = None) -> torch.Tensor:
    """Attention of a step's new tokens over the cache, which holds their own keys and values already.

    q: (B, Hq, N, D), Hq a multiple of the cache's heads. table: (R, M) int32, lens: (R,) int32 tokens of each
    request with its new ones (``Plan.lens``), cu: (R + 1,) int32 the requests' first tokens in q (``Plan.cu``);
    without it every request has B N / R tokens. A request's new tokens are its last ones: the one at
    position p attends to positions <= p, with ``slide_size`` W > 0 only to those > p - W, without ``causal``
    (cross attention) to all of them. Positions whose table entry is no block are not attended to. A row that
    attends to nothing is 0, and so are rows of no request (ahead of ``cu[0]``, from ``cu[R]`` on).

    ``max_new``: the most new tokens of any request, if known (1 for a decoding step): it only chooses
    kernels. ``scale`` defaults to 1/sqrt(D); ``softcap`` as in ``flash_attn_gqa_train``. There is no gradient."""
    _refuse_gradients("attention over the cache", q, q)
    if max_new is not None and max_new < 1:
        raise ValueError("max_new must be at least 1")
    fn = _lib.native().kv4_attention if _plain(q) else torch.ops.gfa.kv4_attention
    return fn(q, cache.codes, cache.scales, cache.dtype is torch.bfloat16, table, lens, cu, max_new or 0, bool(causal),
              int(slide_size or 0), _default_scale(q.shape[-1], scale), _check_softcap(softcap))


# The same calls as registered ops (torch.compile traces them without a break).

@torch.library.custom_op("gfa::kv4_plan", mutates_args=("table",))
def _plan_op(lens: torch.Tensor, new: torch.Tensor, table: torch.Tensor, free: torch.Tensor, used: torch.Tensor,
             block_size: int, tokens: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return _lib.native().kv4_plan(lens, new, table, free, used, block_size, tokens, True)


@_plan_op.register_fake
def _plan_fake(lens, new, table, free, used, block_size, tokens):
    return (lens.new_empty((tokens,), dtype=torch.int64), lens.new_empty((tokens,)), lens.new_empty((lens.shape[0] + 1,)),
            lens.new_empty(lens.shape), lens.new_empty((1,)))


@torch.library.custom_op("gfa::kv4_write", mutates_args=("codes", "scales"))
def _write_op(codes: torch.Tensor, scales: torch.Tensor, bf16: bool, k: torch.Tensor, v: torch.Tensor,
              slots: torch.Tensor) -> None:
    _lib.native().kv4_write(codes, scales, bf16, k, v, slots)


@_write_op.register_fake
def _write_fake(codes, scales, bf16, k, v, slots):
    return None


@torch.library.custom_op("gfa::kv4_read", mutates_args=())
def _read_op(codes: torch.Tensor, scales: torch.Tensor, bf16: bool, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return _lib.native().kv4_read(codes, scales, bf16, slots, True)


@_read_op.register_fake
def _read_fake(codes, scales, bf16, slots):
    H, D, T = codes.shape[1], 2 * codes.shape[4], slots.shape[0]
    k, v = (codes.new_empty((T, H, D), dtype=torch.bfloat16 if bf16 else torch.float16)[None].transpose(1, 2) for _ in range(2))
    return k, v


@torch.library.custom_op("gfa::kv4_attention", mutates_args=())
def _attention_op(q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, bf16: bool, table: torch.Tensor,
                  lens: torch.Tensor, cu: Optional[torch.Tensor], max_new: int, causal: bool, window: int, scale: float,
                  softcap: float) -> torch.Tensor:
    return _lib.native().kv4_attention(q, codes, scales, bf16, table, lens, cu, max_new, causal, window, scale, softcap)


@_attention_op.register_fake
def _attention_fake(q, codes, scales, bf16, table, lens, cu, max_new, causal, window, scale, softcap):
    return _out_like(q)
