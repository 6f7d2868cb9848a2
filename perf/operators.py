"""The serving operators this framework is timed on: a key/value cache held in 4 bits.

A case is one call of a serving step. Its ``op``:

  plan    block tables and slot maps of a step, from the requests' lengths
  store   keys and values of a step's tokens stored in the cache, and read back by their slots
  attend  attention of the step's new tokens over the cache, their own keys and values in it

Keys of a case: B requests; ``ctx`` the longest request's tokens and ``least`` the shortest's share of them; ``new`` the most
new tokens of a request; ``mix``: 0 every request has ``new``, 1 the first has ``new`` and the others one, 2 any number from
one to ``new``; bs tokens per block; Hq, Hkv, D, window, softcap, dtype the attention layer; ``pad`` tokens of padding behind
the last request's. Lengths follow from the case, contents from the seed.

The format: 32 neighbouring channels of a token and head share a power of two (one byte, biased by 127); an element is a
sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6, two to a byte, the even channel in the low bits. Bytes lie in the order in which
a wave's lanes take them, in tiles of 32 tokens (``_places`` below).
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16}
_LOW, _HIGH = {"bf16": -125, "fp16": -23}, {"bf16": 125, "fp16": 13}
_MOST_FLOPS, _MOST_BYTES, _MOST_SCORES = 4.0e12, 6.0e8, 2.2e9


def _case(op, B, ctx, new, Hq=8, Hkv=1, D=512, bs=64, least=1.0, mix=0, window=0, softcap=0.0, dtype="bf16", pad=0, **kw):
    return dict(kw, op=op, B=B, ctx=ctx, new=new, Hq=Hq, Hkv=Hkv, D=D, bs=bs, least=least, mix=mix, window=window,
                softcap=softcap, dtype=dtype, pad=pad)


def listed():
    return [
        # One token for each of a small chat server's eight requests: made once per step, latency counts.
        _case("plan", 8, 16384, 1, least=0.02, name="plan_decode_8"),
        # A large step: prompts of unequal length come in for 256 requests, padded to a fixed token count.
        _case("plan", 256, 8192, 128, least=0.05, mix=2, pad=77, name="plan_prompts_256"),
        # The keys and values of one decoding step, a global layer of Gemma-4-E2B.
        _case("store", 16, 2000, 1, Hkv=1, D=512, least=0.1, name="store_decode_16"),
        # A 16k prompt through the sliding layer of the 16-head model (8 KV heads).
        _case("store", 1, 16384, 16384, Hq=16, Hkv=8, D=256, name="store_prompt_16k"),
        # Prompts of unequal length, a Llama-shaped layer in fp16, with padding.
        _case("store", 5, 4099, 1021, Hq=32, Hkv=8, D=128, least=0.3, mix=2, dtype="fp16", pad=13, name="store_prompts_fp16"),
        # One token of a short chat, Gemma-4-E2B's sliding layer: the smallest attention, 28 times per token.
        _case("attend", 1, 333, 1, Hq=8, Hkv=1, D=256, window=512, name="decode_short_sliding"),
        # One token of a long chat, the same model's global layer: few rows, a long axis.
        _case("attend", 1, 16384, 1, Hq=8, Hkv=1, D=512, name="decode_16k_global"),
        # A batch of 32 requests of very unequal length, the larger model's global layer (32:4).
        _case("attend", 32, 8192, 1, Hq=32, Hkv=4, D=512, least=0.03, name="decode_ragged_32"),
        # A full server: 64 requests, a Llama-shaped layer (32:8), long contexts. Memory's rate counts.
        _case("attend", 64, 16000, 1, Hq=32, Hkv=8, D=128, least=0.4, name="decode_full_64"),
        # Four drafted tokens verified at once, soft-capped logits, fp16, a few requests.
        _case("attend", 6, 3001, 4, Hq=8, Hkv=4, D=256, softcap=50.0, least=0.2, dtype="fp16", name="verify_softcap_fp16"),
        # A prompt's chunk beside seven decoding requests, the sliding layer of the 16-head model (16:8, window 1024).
        _case("attend", 8, 8192, 1000, Hq=16, Hkv=8, D=256, window=1024, least=0.2, mix=1, pad=24, name="mixed_sliding_chunk"),
        # The last 4k chunk of a 16k prompt, the larger model's global layer: the largest, bound by products.
        _case("attend", 1, 16384, 4096, Hq=32, Hkv=4, D=512, name="chunk_4k_of_16k_global"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more call of the same ranges: the layers above, blocks of 32 to 256 tokens, 1 to 256 requests."""
    op = rng.choice(["plan", "store", "attend", "attend", "attend", "attend"])
    Hq, Hkv, D, window, softcap = rng.choice([
        (8, 1, 256, 512, 0.0), (8, 1, 512, 0, 0.0), (32, 4, 512, 0, 0.0), (16, 2, 512, 0, 0.0), (16, 8, 256, 1024, 0.0),
        (32, 8, 128, 0, 0.0), (16, 4, 128, 1024, 0.0), (16, 16, 64, 0, 0.0), (32, 8, 64, 0, 0.0), (8, 4, 256, 0, 50.0),
        (8, 4, 256, 4096, 50.0)])
    B = _log_int(rng, 1, 256 if op == "plan" else 64)
    kind = rng.choice(["one", "one", "few", "chunk"])
    new = 1 if kind == "one" else rng.randint(2, 8) if kind == "few" else _log_int(rng, 16, 4096)
    c = _case(op, B, max(new, _log_int(rng, 64, 16384)), new, Hq, Hkv, D, rng.choice([32, 64, 64, 128, 256]),
              rng.choice([1.0, 0.5, 0.1]), 0 if kind == "one" else rng.choice([0, 1, 2]), window, softcap,
              rng.choice(["bf16", "bf16", "fp16"]), rng.choice([0, 0, rng.randint(1, 40)]))
    while c["B"] > 1 and (work(c)["flops"] > _MOST_FLOPS or work(c)["bytes"] > _MOST_BYTES
                          or c["B"] * c["Hkv"] * c["ctx"] * c["D"] > _MOST_SCORES
                          or c["op"] == "attend" and c["B"] * c["Hq"] * c["new"] * c["ctx"] > _MOST_SCORES):
        c["B"] = c["B"] * 3 // 4
    return c


def _lengths(case):
    """(tokens of each request after the step, new tokens among them)."""
    rng = random.Random(131 * case["ctx"] + 17 * case["new"] + case["B"])
    total, new = [], []
    for b in range(case["B"]):
        n = case["new"] if case["mix"] == 0 or b == 0 else 1 if case["mix"] == 1 else rng.randint(1, case["new"])
        least = max(n, int(case["least"] * case["ctx"]))
        total.append(case["ctx"] if b == 0 else rng.randint(least, max(least, case["ctx"])))
        new.append(n)
    return total, new


def _seen(case, total, new):
    """(keys that some new token of a request attends to, attended pairs of one query head)."""
    w = case["window"] or total
    pairs = sum(min(total - new + i + 1, w) for i in range(new))
    return min(total, w + new - 1), pairs


def work(case):
    total, new = _lengths(case)
    T = sum(new) + case["pad"]
    B, D, Hkv, bs = case["B"], case["D"], case["Hkv"], case["bs"]
    row = D + D // 16  # a token's keys and values of one KV head in the cache
    if case["op"] == "plan":
        grown = sum(-(-n // bs) - -(-(n - k) // bs) for n, k in zip(total, new))
        return {"bytes": B * (4 + 4 + 4 + 4 + 4) + 8 * grown + 12 * T, "flops": 0}
    if case["op"] == "store":
        # in: keys, values, slots; the cache written and read; out: keys, values
        return {"bytes": T * (Hkv * (8 * D + 2 * row) + 16), "flops": 0}
    seen = [_seen(case, n, k) for n, k in zip(total, new)]
    blocks = sum(-(-s // bs) for s, _ in seen)
    return {"bytes": sum(s for s, _ in seen) * Hkv * row + 4 * T * case["Hq"] * D + 4 * blocks + 8 * B,
            "flops": 4 * D * case["Hq"] * sum(p for _, p in seen)}


# ---- inputs ----

def _code(x, dtype):
    """(codes 0..15, exponents) of float rows x: (..., D), blocks of 32 channels."""
    y = x.reshape(*x.shape[:-1], -1, 32)
    amax = y.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1)
    e = torch.where(amax > 0, e - 3 + (m > 0.875).to(e.dtype), torch.full_like(e, -1000)).clamp(_LOW[dtype], _HIGH[dtype])
    a = torch.ldexp(y.abs(), -e)
    c = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return (c + 8 * (y < 0)).to(torch.uint8).reshape(x.shape), e[..., 0]


def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def prepare(case, seed):
    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(seed)
    total, new = _lengths(case)
    B, bs, D, Hkv = case["B"], case["bs"], case["D"], case["Hkv"]
    dtype = _DTYPE[case["dtype"]]
    T = sum(new) + case["pad"]
    have = [-(-(n - k) // bs) for n, k in zip(total, new)]
    want = [-(-n // bs) for n in total]
    num_blocks = sum(want) + 3
    width = max(want) + 2
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    order = torch.randperm(num_blocks, generator=g, device=dev).to(torch.int32)  # blocks are handed out in any order
    state = {"case": case, "bs": bs, "T": T}
    if case["op"] == "plan":
        # blocks already held come first in `order`, the rest is the free list
        table = torch.full((B, width), -1, dtype=torch.int32, device=dev)
        row = torch.repeat_interleave(torch.arange(B, device=dev), ints(have).long())
        col = torch.arange(sum(have), device=dev) - torch.repeat_interleave((ints(have).cumsum(0) - ints(have)).long(), ints(have).long())
        table[row, col] = order[:sum(have)]
        used = 2
        free = torch.cat([order[:used], order[sum(have):]])  # two entries handed out before
        return dict(state, lens=ints([n - k for n, k in zip(total, new)]), new=ints(new), table=table, free=free,
                    used=ints([used]))
    table = torch.full((B, width), -1, dtype=torch.int32, device=dev)
    row = torch.repeat_interleave(torch.arange(B, device=dev), ints(want).long())
    col = torch.arange(sum(want), device=dev) - torch.repeat_interleave((ints(want).cumsum(0) - ints(want)).long(), ints(want).long())
    table[row, col] = order[:sum(want)]
    cu = torch.zeros(B + 1, dtype=torch.int32, device=dev)
    cu[1:] = ints(new).cumsum(0)
    state.update(table=table, lens=ints(total), cu=cu, max_new=max(new), max_len=max(total))
    if case["op"] == "store":
        codes = torch.zeros((num_blocks, Hkv, 2, bs, D // 2), dtype=torch.uint8, device=dev)
        scales = torch.zeros((num_blocks, Hkv, 2, bs, D // 32), dtype=torch.uint8, device=dev)
        slots = torch.full((T,), -1, dtype=torch.int64, device=dev)
        t = torch.arange(T - case["pad"], device=dev)
        b = torch.searchsorted(cu[1:].contiguous(), t.to(torch.int32), right=True)
        pos = (ints(total) - ints(new)).long()[b] + t - cu.long()[b]
        slots[:t.numel()] = table[b, pos // bs].long() * bs + pos % bs
        # keys carry a few strong channels, as a model's do
        strong = 1.0 + 5.0 * (torch.rand((Hkv, 1, D), generator=g, device=dev) < 0.03)
        kv = [torch.randn((T, Hkv, D), generator=g, device=dev) for _ in range(2)]
        kv[0] *= strong.transpose(0, 1)
        k, v = (x.to(dtype)[None].transpose(1, 2) for x in kv)  # (1, Hkv, T, D) views of a projection's rows
        return dict(state, codes=codes, scales=scales, slots=slots, k=k, v=v)
    # a cache in use: rows of codes and exponents of normal values, drawn from a pool
    pool = torch.randn((4096, D), generator=g, device=dev) * torch.exp(0.3 * torch.randn((4096, 1), generator=g, device=dev))
    c, e = _code(pool, case["dtype"])
    pool_c, pool_s = c[:, 0::2] | c[:, 1::2] << 4, (e + 127).to(torch.uint8)
    rows = num_blocks * Hkv * 2 * bs
    pick = torch.randint(0, 4096, (rows,), generator=g, device=dev, dtype=torch.int32)
    codes = pool_c[pick].reshape(num_blocks, Hkv, 2, bs, D // 2)
    scales = pool_s[pick].reshape(num_blocks, Hkv, 2, bs, D // 32)
    q = torch.randn((T, case["Hq"], D), generator=g, device=dev).to(dtype)[None].transpose(1, 2)  # (1, Hq, T, D) view
    return dict(state, codes=codes, scales=scales, q=q)


# ---- the plain forms ----

def _places(D, t, d):
    """Where a tile of 32 tokens keeps channel pair d, d + 1 (d even) of token t, and block d // 32's exponent: byte offsets
    (key codes, value codes, key scales, value scales) inside the tile's 16 D bytes of codes and D bytes of scales."""
    half, g, r = t // 16, t % 16 // 4, t % 4
    w = min(D, 128)
    kc = d // w * (16 * w) + t * (w // 2) + d % w // 2
    p, x = d // (D // 16), d % (D // 16)
    if D >= 128:
        vc = x // 8 * 2048 + half * 1024 + (g * 16 + p) * 16 + r * 4 + x % 8 // 2
        ks = t * (D // 32) + d // 32 % 4 * (D // 128) + d // 128
    else:
        vc = (g * 16 + p) * 16 + half * 8 + r * 2 + x // 2
        ks = t * 2 + d // 32
    vs = (g * (D // 32) + d // 32) * 8 + half * 4 + r
    return kc, vc, ks, vs


def _decode(code, scale):
    """float32 values of codes (0..15) with exponent bytes."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=code.device)
    v = torch.ldexp(grid[(code & 7).long()], scale.to(torch.int32) - 127)
    return torch.where(code >= 8, -v, v)


def _plan(s):
    lens, new, table, free, used, bs, T = (s[x] for x in ("lens", "new", "table", "free", "used", "bs", "T"))
    B, M = table.shape
    have, want = (lens + bs - 1) // bs, (lens + new + bs - 1) // bs
    need = want - have
    start = used + need.cumsum(0) - need
    col = torch.arange(M, device=table.device)[None]
    at = start[:, None] + col - have[:, None]
    grows = (col >= have[:, None]) & (col < want[:, None])
    got = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1).long()], -1)
    table.copy_(torch.where(grows, got, table))
    cu = torch.zeros(B + 1, dtype=torch.int32, device=table.device)
    cu[1:] = new.cumsum(0)
    t = torch.arange(T, device=table.device)
    b = torch.searchsorted(cu[1:].contiguous(), t.to(torch.int32), right=True)
    real = b < B
    b = b.clamp(max=B - 1)
    pos = lens.long()[b] + t - cu.long()[b]
    block = table[b, (pos // bs).clamp(max=M - 1)].long()
    slots = torch.where(real & (pos < M * bs) & (block >= 0), block * bs + pos % bs, -1)
    positions = torch.where(real, pos, 0).to(torch.int32)
    return {"slots": slots, "positions": positions, "cu": cu, "lens": lens + new,
            "used": (used + need.sum()).to(torch.int32), "table": table}


def _store(s):
    D, bs, dtype = s["case"]["D"], s["bs"], s["case"]["dtype"]
    T, Hkv = s["T"], s["case"]["Hkv"]
    out = []
    slots = s["slots"]
    real = slots >= 0
    slot = slots[real]
    block, off = slot // bs, slot % bs
    codes, scales = s["codes"].view(-1), s["scales"].view(-1)
    head = torch.arange(Hkv, device=slot.device)[None, :, None]
    d = torch.arange(0, D, 2, device=slot.device)[None, None]
    d32 = torch.arange(0, D, 32, device=slot.device)[None, None]
    for side, x in ((0, s["k"]), (1, s["v"])):
        page = (block[:, None, None] * Hkv + head) * 2 + side
        at = page * (bs * D // 2) + (off // 32)[:, None, None] * (16 * D) + _places(D, (off % 32)[:, None, None], d)[side]
        at_s = page * (bs * D // 32) + (off // 32)[:, None, None] * D + _places(D, (off % 32)[:, None, None], d32)[2 + side]
        c, e = _code(x[0].transpose(0, 1)[real].float(), dtype)
        codes[at] = c[..., 0::2] | c[..., 1::2] << 4
        scales[at_s] = (e + 127).to(torch.uint8)
        byte, e = codes[at], scales[at_s]
        got = _decode(torch.stack([byte & 15, byte >> 4], -1).reshape(-1, Hkv, D), e.repeat_interleave(32, -1))
        y = torch.zeros((T, Hkv, D), dtype=_DTYPE[dtype], device=slot.device)
        y[real] = got.to(y.dtype)
        out.append(y[None].transpose(1, 2))
    return {"k": out[0], "v": out[1]}


def _pages(s, L):
    """float32 keys and values (B, Hkv, L, D) of the requests' first L slots, gathered by the block table."""
    case = s["case"]
    D, bs, Hkv, B = case["D"], s["bs"], case["Hkv"], case["B"]
    n = -(-L // bs)
    ids = s["table"][:, :n].clamp(min=0).long()
    tiles = bs // 32
    c, e = s["codes"][ids], s["scales"][ids]  # (B, n, Hkv, 2, bs, ...)
    c, e = c.reshape(B, n, Hkv, 2, tiles, 16 * D), e.reshape(B, n, Hkv, 2, tiles, D)
    kc, vc, ks, vs = c[:, :, :, 0], c[:, :, :, 1], e[:, :, :, 0], e[:, :, :, 1]
    w = min(D, 128)
    kc = kc.reshape(B, n, Hkv, tiles, D // w, 32, w // 2).transpose(4, 5).reshape(B, n, Hkv, tiles, 32, D // 2)
    if D >= 128:
        vc = vc.reshape(B, n, Hkv, tiles, D // 128, 2, 4, 16, 4, 4).permute(0, 1, 2, 3, 5, 6, 8, 7, 4, 9)
        ks = ks.reshape(B, n, Hkv, tiles, 32, 4, D // 128).transpose(5, 6)
    else:
        vc = vc.reshape(B, n, Hkv, tiles, 4, 16, 2, 4, 2).permute(0, 1, 2, 3, 6, 4, 7, 5, 8)
    vc, ks = vc.reshape(B, n, Hkv, tiles, 32, D // 2), ks.reshape(B, n, Hkv, tiles, 32, D // 32)
    vs = vs.reshape(B, n, Hkv, tiles, 4, D // 32, 2, 4).permute(0, 1, 2, 3, 6, 4, 7, 5).reshape(B, n, Hkv, tiles, 32, D // 32)

    def whole(code, scale):
        v = _decode(torch.stack([code & 15, code >> 4], -1).reshape(*code.shape[:-1], D), scale.repeat_interleave(32, -1))
        return v.reshape(B, n, Hkv, bs, D).transpose(1, 2).reshape(B, Hkv, n * bs, D)[:, :, :L].contiguous()

    return whole(kc, ks), whole(vc, vs)


def _attend(s):
    case = s["case"]
    B, Hq, Hkv, D, T = case["B"], case["Hq"], case["Hkv"], case["D"], s["T"]
    L, N, G = s["max_len"], s["max_new"], Hq // Hkv
    k, v = _pages(s, L)
    cu, lens = s["cu"].long(), s["lens"].long()
    new = cu[1:] - cu[:-1]
    i = torch.arange(N, device=k.device)[None]
    t = (cu[:-1, None] + i).clamp(max=T - 1)
    q = s["q"][0].float()[:, t]  # (Hq, B, N, D)
    q = q.reshape(Hkv, G, B, N, D).permute(2, 0, 1, 3, 4).reshape(B, Hkv, G * N, D).contiguous()
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(D))
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    pos = (lens - new)[:, None] + i  # (B, N)
    j = torch.arange(L, device=k.device)
    ok = (j <= pos[..., None]) & (i < new[:, None])[..., None]
    if case["window"]:
        ok = ok & (j > pos[..., None] - case["window"])
    x = torch.where(ok[:, None, None], x.reshape(B, Hkv, G, N, L), -math.inf)
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    norm = x.sum(-1, keepdim=True)
    o = torch.matmul(x.reshape(B, Hkv, G * N, L), v).reshape(B, Hkv, G, N, D)
    o = torch.where(norm > 0, o / norm, 0.0).permute(0, 3, 1, 2, 4).reshape(B, N, Hq, D)
    real = i < new[:, None]
    out = torch.zeros((T, Hq, D), dtype=s["q"].dtype, device=k.device)
    out[t[real]] = o[real].to(out.dtype)
    return out[None].transpose(1, 2)


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"plan": _plan, "store": _store, "attend": _attend}[op](state)
    from gemma_triton_flash_attn_amd import kv4

    s, case = state, state["case"]
    if op == "plan":
        p = kv4.plan(s["lens"], s["new"], s["table"], s["free"], s["used"], block_size=s["bs"], tokens=s["T"])
        return {"slots": p.slots, "positions": p.positions, "cu": p.cu, "lens": p.lens, "used": p.used, "table": s["table"]}
    cache = kv4.Cache(s["codes"], s["scales"], _DTYPE[case["dtype"]])
    if op == "store":
        kv4.write(cache, s["k"], s["v"], s["slots"])
        k, v = kv4.read(cache, s["slots"])
        return {"k": k, "v": v}
    return kv4.attention(s["q"], cache, s["table"], s["lens"], s["cu"], max_new=s["max_new"], slide_size=case["window"],
                         softcap=case["softcap"] or None)


# ---- the definition in 64 bits ----

def _exact_store(s):
    low, high = _LOW[s["case"]["dtype"]], _HIGH[s["case"]["dtype"]]
    real = (s["slots"] >= 0)[None, None, :, None]
    out = {}
    for name in ("k", "v"):
        x = s[name].double()
        y = x.unflatten(-1, (-1, 32))
        top = y.abs().amax(-1, keepdim=True)
        e = torch.floor(torch.log2(top.clamp(min=2.0 ** -140))) - 2
        e = (e + (top > 7 * torch.exp2(e))).clamp(low, high)
        a = y.abs() / torch.exp2(e)
        # the grid is even inside [0, 2], [2, 4] and [4, 8]; round() takes ties to even, as the codes do
        a = torch.where(a < 2, torch.round(2 * a) / 2, torch.where(a < 4, torch.round(a), 2 * torch.round(a / 2))).clamp(max=6)
        out[name] = torch.where(real, (torch.sign(y) * a * torch.exp2(e)).flatten(-2), 0.0)
    return out


def _exact_attend(s):
    case = s["case"]
    D, Hq, Hkv, bs, w, cap = case["D"], case["Hq"], case["Hkv"], s["bs"], case["window"], case["softcap"]
    G = Hq // Hkv
    cu, lens, table = s["cu"].tolist(), s["lens"].tolist(), s["table"].long()
    out = torch.zeros((s["T"], Hq, D), dtype=torch.float64, device=table.device)
    codes, scales = s["codes"].view(-1), s["scales"].view(-1)
    d = torch.arange(D, device=table.device)[None]

    def rows(side, h, slot):
        page, tile, t = ((slot // bs) * Hkv + h) * 2 + side, slot % bs // 32, (slot % 32)[:, None]
        byte = codes[(page * (bs * D // 2) + tile * (16 * D))[:, None] + _places(D, t, d - d % 2)[side]].int()
        e = scales[(page * (bs * D // 32) + tile * D)[:, None] + _places(D, t, d - d % 32)[2 + side]].double() - 127
        c = torch.where(d % 2 == 1, byte >> 4, byte & 15)
        n = c & 7
        size = torch.where(n < 2, n * 0.5, (1 + 0.5 * (n & 1)) * torch.exp2((n >> 1).double() - 1))
        return torch.where(c > 7, -size, size) * torch.exp2(e)

    for b in range(case["B"]):
        n, new, t0 = lens[b], cu[b + 1] - cu[b], cu[b]
        first = max(0, n - new - w + 1) if w else 0
        j = torch.arange(first, n, device=table.device)
        slot = table[b, j // bs] * bs + j % bs
        p = torch.arange(n - new, n, device=table.device)[:, None]
        hidden = (j[None] > p) | ((j[None] <= p - w) if w else False)
        for h in range(Hkv):
            k, v = rows(0, h, slot), rows(1, h, slot)
            for a in range(G):
                x = s["q"][0, h * G + a, t0:t0 + new].double() @ k.t().contiguous() / math.sqrt(D)
                x = cap * torch.tanh(x / cap) if cap else x
                out[t0:t0 + new, h * G + a] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v
    return out[None].transpose(1, 2)


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    return _exact_store(s) if case["op"] == "store" else _exact_attend(s)
