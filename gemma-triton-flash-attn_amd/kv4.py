"""Serving: attention over a key/value cache held in 4 bits, for requests that may share what they have in common.

The rest of the framework attends the tokens of one call to each other. A server that generates text
attends each step's new tokens to everything before them. This module keeps those keys and values in
4.25 bits per element, in blocks that requests of unequal length take from one pool:

    cache = kv4.allocate(num_blocks, heads_kv, head_dim)            # one per layer
    step = kv4.plan(lens, new, table, free, used, block_size=cache.block_size, tokens=T)
    kv4.write(cache, k, v, step.slots)                              # the step's keys and values, stored
    o = kv4.attention(q, cache, table, step.lens, step.cu)          # its queries over all of the cache

    f = kv4.fork(caches, table, lens, free, used, parents=parents)  # several answers to one prompt, beams: shared blocks
    shared = kv4.share(table, step.lens, step.cu, block_size=cache.block_size)        # what they have in common
    o = kv4.attention(q, cache, table, step.lens, step.cu, max_new=1, shared=shared)  # read once for all of them
    v = kv4.verify(target, draft, tokens, accept, sample, step.lens, step.cu)         # drafted tokens of a step
    f = kv4.fork(caches, table, step.lens, free, step.used, keep=v.lens)              # those not accepted taken back

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

from typing import NamedTuple, Optional, Sequence, Union

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


class Shared(NamedTuple):
    """What requests of a step have in common (``share``)."""

    skip: torch.Tensor  # (requests,) int32: tokens of the request's prefix
    cu: torch.Tensor    # (requests + 1,) int32: first tokens of the groups, each taken as one request
    lens: torch.Tensor  # (requests,) int32: tokens of a group's prefix, where its first request stands


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
              softcap: Optional[float] = None, shared: Optional[Shared] = None, apart: bool = False) -> torch.Tensor:
    """Attention of a step's new tokens over the cache, which holds their own keys and values already.

    q: (B, Hq, N, D), Hq a multiple of the cache's heads. table: (R, M) int32, lens: (R,) int32 tokens of each
    request with its new ones (``Plan.lens``), cu: (R + 1,) int32 the requests' first tokens in q (``Plan.cu``);
    without it every request has B N / R tokens. A request's new tokens are its last ones: the one at
    position p attends to positions <= p, with ``slide_size`` W > 0 only to those > p - W, without ``causal``
    (cross attention) to all of them. Positions whose table entry is no block are not attended to. A row that
    attends to nothing is 0, and so are rows of no request (ahead of ``cu[0]``, from ``cu[R]`` on).

    ``max_new``: the most new tokens of any request, if known (1 for a decoding step): it only chooses
    kernels. ``scale`` defaults to 1/sqrt(D); ``softcap`` as in ``flash_attn_gqa_train``. There is no gradient.

    ``shared``: ``share``'s result for this table, lens and cu. The prefix of a group of requests is then read once for all
    of them, and the parts are joined: the same result within the same bound, with other roundings (weights are rounded to
    16 bits against a maximum of their part, which below head dim 512 is exact without ``shared`` and may be passed by 2^8
    in a prefix, and 32-bit sums are taken in another order). That is done where the lengths of all requests promise that
    it is faster, which is found on the device, or with ``apart`` wherever there is a group. Tables too narrow to gain by it
    take the call without ``shared``; in wide ones, whose requests' lengths the host does not know, a call that finds little
    in common can take some us longer than without.

    It has no effect with ``slide_size``, nor where requests have many query rows (``max_new``, else the average, times
    Hq / Hkv above 64; 128 where requests times KV heads are at most four), which are bound by products; without ``max_new``
    single requests of more rows than that are computed as without ``shared``, beside the others."""
    _refuse_gradients("attention over the cache", q, q)
    if max_new is not None and max_new < 1:
        raise ValueError("max_new must be at least 1")
    fn = _lib.native().kv4_attention if _plain(q) else torch.ops.gfa.kv4_attention
    return fn(q, cache.codes, cache.scales, cache.dtype is torch.bfloat16, table, lens, cu, max_new or 0, bool(causal),
              int(slide_size or 0), _default_scale(q.shape[-1], scale), _check_softcap(softcap),
              *(shared if shared is not None else (None, None, None)), bool(apart))


class Fork(NamedTuple):
    """Block tables after ``fork``."""

    table: torch.Tensor  # (rows, M) int32
    lens: torch.Tensor   # (rows,) int32: tokens of each row
    used: torch.Tensor   # (1,) int32: entries of the free list handed out


class Compact(NamedTuple):
    """Block tables after ``compact``."""

    table: torch.Tensor  # (requests, M) int32
    used: torch.Tensor   # (1,) int32: blocks that requests hold, the first ones of the pool


class Verified(NamedTuple):
    """A step's tokens after ``verify``."""

    tokens: torch.Tensor    # (tokens,) int64: what follows each token of the step: accepted ones, the drawn one, -1 behind it
    accepted: torch.Tensor  # (requests,) int32: drafted tokens accepted
    lens: torch.Tensor      # (requests,) int32: tokens whose keys and values are worth keeping


def _arrays(caches: Union[Cache, Sequence[Cache]]) -> tuple[list[torch.Tensor], list[torch.Tensor]]:
    caches = [caches] if isinstance(caches, Cache) else list(caches)
    if not caches:
        raise ValueError("at least one cache is needed")
    return [c.codes for c in caches], [c.scales for c in caches]


def fork(caches: Union[Cache, Sequence[Cache]], table: torch.Tensor, lens: torch.Tensor, free: torch.Tensor, used: torch.Tensor, *,
         parents: Optional[torch.Tensor] = None, keep: Optional[torch.Tensor] = None) -> Fork:
    """The block tables of the next step's requests, from this one's: several answers to one prompt, beams that go on or are
    dropped, requests that left, tokens taken back.

    caches: the layers' caches that the table is of, one num_blocks (at most 2^18) and block size. table: (B, M) int32, lens: (B,)
    int32 tokens of each request; every block of the pool that some request holds has to be in it, the first ceil(lens /
    block_size) entries of a row. parents: (rows,) int32, the request that each row goes on from; anything but 0 .. B - 1 an
    empty row; default: row r from request r. keep: (rows,) int32, tokens that it keeps at most; default: all. B and rows
    at most 4096.

    Rows share their parents' blocks. A row writes its next tokens behind its last one, so a block that it keeps only a part of
    has to be its own: it stays with the first such row if no row keeps it whole, and is copied for the others, in every cache.
    Blocks that no row holds any more are given back, in ascending order in front of ``used`` in the free list (free: (F,) int32,
    contiguous, changed in place: an entry for every block that was ever taken from it). Copies take those first, then entries from ``used``
    ((1,) int32) on. Where the list ends, the row's entry is -1 and ``Fork.used`` above F tells of it. The inputs but for free and the
    caches are only read. Results are views of one allocation outside of torch.compile."""
    codes, scales = _arrays(caches)
    if _plain(table):
        return Fork(*_lib.native().kv4_fork(codes, scales, table, lens, free, used, parents, keep, False))
    return Fork(*torch.ops.gfa.kv4_fork(codes, scales, table, lens, free, used, parents, keep))


def compact(caches: Union[Cache, Sequence[Cache]], table: torch.Tensor, lens: torch.Tensor, free: torch.Tensor) -> Compact:
    """Moves the blocks that requests hold to the lowest ids of the pool, so that the rest of it can be given up or used otherwise.

    caches, table and lens as in ``fork``. Of n blocks held, the k-th (in ascending order) at or past n goes to the k-th id below n that
    nobody holds, in every cache. free: (num_blocks,) int32, all of the pool, contiguous; becomes 0, 1, 2, ... in place, its first
    ``Compact.used`` entries handed out."""
    codes, scales = _arrays(caches)
    if _plain(table):
        return Compact(*_lib.native().kv4_compact(codes, scales, table, lens, free, False))
    return Compact(*torch.ops.gfa.kv4_compact(codes, scales, table, lens, free))


def copy(caches: Union[Cache, Sequence[Cache]], src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copies block ``src[i]`` to block ``dst[i]`` ((pairs,) int32) in every cache; pairs with an id that is no block are left
    out. No block may be the destination of two pairs, or of one and the source of another."""
    codes, scales = _arrays(caches)
    (_lib.native().kv4_copy if _plain(src) else torch.ops.gfa.kv4_copy)(codes, scales, src, dst)


def share(table: torch.Tensor, lens: torch.Tensor, cu: torch.Tensor, *, block_size: int, least: int = 512) -> Shared:
    """What a step's requests have in common, for ``attention``'s ``shared``: once per step, for all layers.

    table: (R, M) int32, lens: (R,) int32 tokens with the new ones (``Plan.lens``), cu: (R + 1,) int32 (``Plan.cu``). Requests next to
    each other whose rows begin with the same blocks, at least ``least`` tokens of them (a row's blocks that are full ahead of its new
    tokens count), form a group; its prefix is what any two neighbours in it have in common. So answers to one prompt
    should stand side by side, and where all requests begin with the same short text ``least`` above its length keeps
    their prompts apart. At most 4096 requests. Results are views of one allocation outside of torch.compile."""
    if _plain(table):
        return Shared(*_lib.native().kv4_share(table, lens, cu, block_size, least, False))
    return Shared(*torch.ops.gfa.kv4_share(table, lens, cu, block_size, least))


def verify(target: torch.Tensor, draft: Optional[torch.Tensor], tokens: torch.Tensor, accept: torch.Tensor, sample: torch.Tensor,
           lens: torch.Tensor, cu: Optional[torch.Tensor] = None) -> Verified:
    """Which of a step's drafted tokens to keep, and the token that follows them: distributed as the target's whatever the draft.

    A request's tokens of the step are its last known one and the drafted ones (packed as for ``attention``: cu (R + 1,) int32, or
    T / R each). target: (T, V), probabilities in fp32, fp16 or bf16: row t what the target gives for the token after token t. draft:
    (T, V) of the same type, row t what token t was drawn from (a request's first row is not read); None where tokens were proposed
    for certain. tokens: (T,) int64. accept: (T,), sample: (R,) float32, uniform in [0, 1), drawn by the caller. Strided rows are read in place.

    Token t is accepted, in order, while accept[t] * draft[t, x] < target[t - 1, x], x = tokens[t] (compared exactly). Then one token
    is drawn: where a drafted one was not accepted from max(target - draft, 0), else from the target, as the first entry at which the
    running sum of weights (64 bits) exceeds sample times their sum. A request without drafted tokens is sampled. Where
    target and draft leave no weight, the target's probabilities are taken; without any of those the token is -1. Values that are no
    finite positive number count as 0.

    lens: (R,) int32 (``Plan.lens``); ``Verified.lens`` is less the tokens not accepted, which ``fork``'s ``keep`` takes back; outside of
    torch.compile it shares an allocation with ``accepted``. There is no gradient."""
    _refuse_gradients("verification", target, target if draft is None else draft)
    if _plain(target):
        return Verified(*_lib.native().kv4_verify(target, draft, tokens, accept, sample, lens, cu, False))
    return Verified(*torch.ops.gfa.kv4_verify(target, draft, tokens, accept, sample, lens, cu))


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
                  softcap: float, shared_skip: Optional[torch.Tensor] = None, shared_cu: Optional[torch.Tensor] = None,
                  shared_lens: Optional[torch.Tensor] = None, apart: bool = False) -> torch.Tensor:
    return _lib.native().kv4_attention(q, codes, scales, bf16, table, lens, cu, max_new, causal, window, scale, softcap,
                                       shared_skip, shared_cu, shared_lens, apart)


@_attention_op.register_fake
def _attention_fake(q, codes, scales, bf16, table, lens, cu, max_new, causal, window, scale, softcap, shared_skip=None,
                    shared_cu=None, shared_lens=None, apart=False):
    return _out_like(q)


@torch.library.custom_op("gfa::kv4_fork", mutates_args=("codes", "scales", "free"))
def _fork_op(codes: Sequence[torch.Tensor], scales: Sequence[torch.Tensor], table: torch.Tensor, lens: torch.Tensor, free: torch.Tensor,
             used: torch.Tensor, parents: Optional[torch.Tensor], keep: Optional[torch.Tensor]
             ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _lib.native().kv4_fork(codes, scales, table, lens, free, used, parents, keep, True)


@_fork_op.register_fake
def _fork_fake(codes, scales, table, lens, free, used, parents, keep):
    rows = (lens if parents is None else parents).shape[0]
    return table.new_empty((rows, table.shape[1])), lens.new_empty((rows,)), lens.new_empty((1,))


@torch.library.custom_op("gfa::kv4_compact", mutates_args=("codes", "scales", "free"))
def _compact_op(codes: Sequence[torch.Tensor], scales: Sequence[torch.Tensor], table: torch.Tensor, lens: torch.Tensor,
                free: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return _lib.native().kv4_compact(codes, scales, table, lens, free, True)


@_compact_op.register_fake
def _compact_fake(codes, scales, table, lens, free):
    return table.new_empty(table.shape), lens.new_empty((1,))


@torch.library.custom_op("gfa::kv4_copy", mutates_args=("codes", "scales"))
def _copy_op(codes: Sequence[torch.Tensor], scales: Sequence[torch.Tensor], src: torch.Tensor, dst: torch.Tensor) -> None:
    _lib.native().kv4_copy(codes, scales, src, dst)


@_copy_op.register_fake
def _copy_fake(codes, scales, src, dst):
    return None


@torch.library.custom_op("gfa::kv4_share", mutates_args=())
def _share_op(table: torch.Tensor, lens: torch.Tensor, cu: torch.Tensor, block_size: int, least: int
              ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _lib.native().kv4_share(table, lens, cu, block_size, least, True)


@_share_op.register_fake
def _share_fake(table, lens, cu, block_size, least):
    return lens.new_empty(lens.shape), lens.new_empty(cu.shape), lens.new_empty(lens.shape)


@torch.library.custom_op("gfa::kv4_verify", mutates_args=())
def _verify_op(target: torch.Tensor, draft: Optional[torch.Tensor], tokens: torch.Tensor, accept: torch.Tensor, sample: torch.Tensor,
               lens: torch.Tensor, cu: Optional[torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _lib.native().kv4_verify(target, draft, tokens, accept, sample, lens, cu, True)


@_verify_op.register_fake
def _verify_fake(target, draft, tokens, accept, sample, lens, cu):
    return tokens.new_empty(tokens.shape), lens.new_empty(lens.shape), lens.new_empty(lens.shape)
