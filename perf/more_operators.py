"""The serving operators this framework is timed on where requests have something in common: answers to one prompt over one
set of cache blocks, tokens that were drafted and have to be verified.

A case is one call of a serving step. Its ``op``:

  share    what neighbouring requests' block tables have in common, once per step
  attend   attention of the step's new tokens over the 4-bit cache, a group's common prefix computed once
  fork     block tables of the next step's requests from this one's (new answers, beams, tokens taken back): blocks shared,
           copied where two requests would write to one, given back where none holds them
  compact  a pool's live blocks moved to its lowest ids
  verify   drafted tokens accepted or not by the target's probabilities, and the token that follows them

Keys of a case. share and attend: ``groups`` prompts with ``answers`` requests each, ``prompt`` tokens of the longest prompt and
``least`` the shortest's share of them, up to ``own`` further tokens of a request, ``new`` tokens each in this step; bs tokens
per block; Hq, Hkv, D, softcap, dtype the attention layer. fork and compact: the same requests as rows of the table; ``how`` they are
forked; L layers of Hkv heads of D channels; ``spare`` blocks of the pool that no request holds. verify: R requests with up to
``drafts`` drafted tokens, V tokens of the vocabulary; ``sure``: the draft gives tokens and no probabilities. Lengths follow from the
case, contents from the seed.

The cache's format is the framework's MXFP4: 32 neighbouring channels of a token and head share a power of two (one byte, biased
by 127); an element is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6, two to a byte. Bytes lie in the order in which a wave's
lanes take them, in tiles of 32 tokens (``_pages`` and ``_rows`` below). Pages are moved as they are: their bytes are the outputs.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_LOW, _HIGH = {"bf16": -125, "fp16": -23}, {"bf16": 125, "fp16": 13}
_LEAST = 512  # tokens that neighbours have in common before they are a group
_MOST_BYTES, _MOST_FLOPS, _MOST_GATHERED = 1.3e9, 5.0e10, 1.2e9


def _case(op, groups=1, answers=4, prompt=1000, least=1.0, own=100, new=1, bs=64, Hq=8, Hkv=1, D=256, softcap=0.0,
          dtype="bf16", **kw):
    return dict(kw, op=op, groups=groups, answers=answers, prompt=prompt, least=least, own=own, new=new, bs=bs, Hq=Hq, Hkv=Hkv,
                D=D, softcap=softcap, dtype=dtype)


def _verified(R, drafts, V, sure=False, dtype="fp32", **kw):
    return dict(kw, op="verify", R=R, drafts=drafts, V=V, sure=sure, dtype=dtype)


def listed():
    return [
        # Eight answers to one 16k prompt, the smallest plan of sharing: made once per step, latency counts.
        _case("share", 1, 8, 16384, name="share_8"),
        # A full server: 32 prompts of unequal length with eight answers each.
        _case("share", 32, 8, 8192, 0.1, 2000, name="share_256"),
        # Four answers to a short question, Gemma-4-E2B's global layer: the smallest attention.
        _case("attend", 1, 4, 700, 1.0, 150, Hq=8, Hkv=1, D=512, name="answers_4_short"),
        # 64 sampled answers to one long prompt, a Llama-shaped layer (32:8).
        _case("attend", 1, 64, 16384, 1.0, 600, Hq=32, Hkv=8, D=128, name="answers_64_of_16k"),
        # Four prompts of unequal length, eight answers each, the larger model's global layer (32:4).
        _case("attend", 4, 8, 8192, 0.3, 1000, Hq=32, Hkv=4, D=512, name="answers_8_of_4_prompts"),
        # Sixteen answers whose four drafted tokens are verified at once, soft-capped logits, fp16, odd lengths.
        _case("attend", 1, 16, 3001, 1.0, 333, 4, Hq=8, Hkv=4, D=256, softcap=50.0, dtype="fp16", name="drafts_16_softcap_fp16"),
        # Eight beams, some dropped and some continued twice, four layers.
        _case("fork", 1, 8, 1000, 1.0, 300, Hkv=1, D=256, how="beams", L=4, spare=64, name="fork_beams_8"),
        # 24 prompts that get eight answers each, a Llama-shaped model of eight layers.
        _case("fork", 24, 1, 4099, 0.2, 1, Hkv=8, D=128, how="answers", L=8, spare=400, name="fork_24_prompts_8"),
        # A small pool half empty.
        _case("compact", 3, 2, 900, 0.4, 200, Hkv=1, D=256, L=2, spare=60, name="compact_small"),
        # A server's pool after its long requests left, four layers: memory's rate counts.
        _case("compact", 40, 2, 5003, 0.1, 500, Hkv=8, D=128, L=4, spare=2500, name="compact_pool"),
        # Four drafted tokens of each of a small server's eight requests.
        _verified(8, 4, 32000, name="verify_8"),
        # 64 requests with up to six drafted tokens, a large vocabulary.
        _verified(64, 6, 262144, name="verify_64_large"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more call of the same ranges: the layers above, 1 to 256 requests, blocks of 32 to 256 tokens."""
    op = rng.choice(["share", "attend", "attend", "attend", "fork", "fork", "compact", "verify", "verify"])
    if op == "verify":
        return _verified(_log_int(rng, 1, 64), rng.choice([0, 1, 3, 4, 7]), _log_int(rng, 1000, 262144),
                         rng.choice([False, False, True]), rng.choice(["fp32", "fp32", "bf16", "fp16"]))
    Hq, Hkv, D, softcap = rng.choice([(8, 1, 256, 0.0), (8, 1, 512, 0.0), (32, 4, 512, 0.0), (16, 8, 256, 0.0), (32, 8, 128, 0.0),
                                      (16, 16, 64, 0.0), (8, 4, 256, 50.0), (16, 2, 64, 30.0)])
    c = _case(op, _log_int(rng, 1, 16), _log_int(rng, 1, 64), _log_int(rng, 64, 16384), rng.choice([1.0, 0.5, 0.1]),
              _log_int(rng, 1, 2000), rng.choice([1, 1, 1, 2, 5, 8]), rng.choice([32, 64, 64, 128, 256]), Hq, Hkv, D, softcap,
              rng.choice(["bf16", "bf16", "fp16"]))
    if op in ("fork", "compact"):
        c.update(how=rng.choice(["beams", "answers", "taken_back"]), L=rng.choice([1, 2, 4, 8]), spare=_log_int(rng, 8, 1000))
    if op == "share":
        c.update(answers=max(2, c["answers"]), prompt=max(1200, c["prompt"]))
    while c["groups"] * c["answers"] > 1 and _too_large(c):
        c["groups" if c["groups"] >= c["answers"] else "answers"] -= max(1, max(c["groups"], c["answers"]) // 4)
    while _too_large(c):
        c["prompt"], c["own"], c["L"] = max(64, c["prompt"] // 2), max(1, c["own"] // 2), max(1, c.get("L", 1) // 2)
    return c


def _too_large(c):
    w = work(c)
    total = _lengths(c)[1]
    if c["op"] in ("fork", "compact"):  # the pool itself
        pool = (sum(-(-n // c["bs"]) for n in total) + c["spare"]) * c["bs"] * c["Hkv"] * (c["D"] + c["D"] // 16) * c["L"]
        return pool > 3.0e9 or w["bytes"] > _MOST_BYTES
    return (w["bytes"] > _MOST_BYTES or w["flops"] > _MOST_FLOPS
            or len(total) * c["Hkv"] * max(total) * c["D"] > _MOST_GATHERED)


def _lengths(case):
    """(tokens of each prompt, tokens of each request with the step's new ones), requests of a prompt side by side."""
    rng = random.Random(131 * case["prompt"] + 17 * case["own"] + case["groups"])
    prompts, total = [], []
    for g in range(case["groups"]):
        least = max(1, int(case["least"] * case["prompt"]))
        prompts.append(case["prompt"] if g == 0 else rng.randint(least, case["prompt"]))
        total += [prompts[-1] + rng.randint(0, case["own"]) + case["new"] for _ in range(case["answers"])]
    return prompts, total


def _parents(case, total):
    """(row of each new request, tokens that it keeps): lists."""
    rng, B = random.Random(len(total) + total[0]), len(total)
    if case["how"] == "beams":  # each of a prompt's beams continues one of them
        n = case["answers"]
        parents = [b // n * n + rng.randrange(n) for b in range(B)]
        return parents, [total[p] for p in parents]
    if case["how"] == "answers":  # eight answers to each, the first tokens of one in four left out
        parents = [b for b in range(B) for _ in range(8)]
        return parents, [total[p] if rng.random() < 0.75 else total[p] - min(total[p], rng.randint(0, 40)) for p in parents]
    return list(range(B)), [n - rng.randint(0, min(n, 8)) for n in total]  # drafted tokens taken back


def _draft_counts(case):
    rng = random.Random(case["V"] + 7 * case["R"] + case["drafts"])
    return [rng.randint(0, case["drafts"]) if b else case["drafts"] for b in range(case["R"])]


def _forked(case):
    """(blocks that requests hold before, blocks copied): as many as the definition gives, contents aside."""
    prompts, total = _lengths(case)
    rows = _block_names(case, prompts, total)
    parents, keep = _parents(case, total)
    bs, whole, part = case["bs"], set(), []
    for p, n in zip(parents, keep):
        whole.update(rows[p][: n // bs])
        if n % bs:
            part.append(rows[p][n // bs])
    first, copies = set(), 0
    for x in part:
        copies += x in whole or x in first
        first.add(x)
    return sum(len(r) for r in rows), copies


def _block_names(case, prompts, total):
    """Blocks of each request by position, as numbers from 0 on: a prompt's whole blocks are its answers' together."""
    rows, nxt, bs, n = [], 0, case["bs"], case["answers"]
    for g, prompt in enumerate(prompts):
        common = list(range(nxt, nxt + (prompt // bs if n > 1 else 0)))
        nxt += len(common)
        for t in total[g * n:(g + 1) * n]:
            k = -(-t // bs) - len(common)
            rows.append(common + list(range(nxt, nxt + k)))
            nxt += k
    return rows


def work(case):
    if case["op"] == "verify":
        # the target's and the draft's row that the next token comes from, a probability of each drafted token, the numbers
        R, size = case["R"], 2 if case["dtype"] != "fp32" else 4
        T = sum(_draft_counts(case)) + R
        rows = 1 if case["sure"] else 2
        return {"bytes": R * case["V"] * size * rows + T * (8 + 8 + 4 + 2 * size) + R * 20, "flops": 3 * R * case["V"]}
    prompts, total = _lengths(case)
    B, bs, D, Hkv = len(total), case["bs"], case["D"], case["Hkv"]
    row = D + D // 16  # a token's keys and values of one KV head in the cache
    n = case["answers"]
    if case["op"] == "share":
        return {"bytes": sum(4 * -(-t // bs) for t in total) + 4 * (2 * B + 1) + 4 * (3 * B + 1), "flops": 0}
    if case["op"] == "attend":
        read = sum((p // bs * bs if n > 1 and p // bs * bs >= _LEAST else 0) for p in prompts)
        read += sum(t - (prompts[b // n] // bs * bs if n > 1 and prompts[b // n] // bs * bs >= _LEAST else 0) for b, t in enumerate(total))
        T = B * case["new"]
        pairs = sum(case["new"] * t - case["new"] * (case["new"] - 1) // 2 for t in total)
        return {"bytes": read * Hkv * row + 4 * T * case["Hq"] * D + sum(4 * -(-t // bs) for t in total) + 8 * B,
                "flops": 4 * D * case["Hq"] * pairs}
    page = case["L"] * bs * Hkv * row
    if case["op"] == "fork":
        held, copies = _forked(case)
        parents, keep = _parents(case, total)
        out = len(parents) * _width(case, total)
        return {"bytes": 4 * (held + out + B + 3 * len(parents)) + 2 * copies * page, "flops": 0}
    names = _block_names(case, prompts, total)
    live = sum(len(set(r)) for r in names) - sum((n - 1) * (p // bs) for p in prompts if n > 1)
    blocks = live + case["spare"]
    # blocks lie anywhere in the pool: a live block is past the live ones' number with the share of spare ones
    moves = live * case["spare"] // blocks
    return {"bytes": 4 * (2 * B * _width(case, total) + B + blocks) + 2 * moves * page, "flops": 0}


def _width(case, total):
    return max(-(-n // case["bs"]) for n in total) + 2


# ---- inputs ----

def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=_dev())


def prepare(case, seed):
    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(seed)
    if case["op"] == "verify":
        return _prepare_verify(case, g)
    prompts, total = _lengths(case)
    names = _block_names(case, prompts, total)
    bs, D, Hkv = case["bs"], case["D"], case["Hkv"]
    live = max(r[-1] for r in names) + 1
    blocks = live + case.get("spare", 3)
    order = torch.randperm(blocks, generator=g, device=dev).to(torch.int32)  # blocks are handed out in any order
    table = torch.full((len(total), _width(case, total)), -1, dtype=torch.int32)
    for b, r in enumerate(names):
        table[b, : len(r)] = torch.tensor(r, dtype=torch.int32)
    table = table.to(dev)
    table = torch.where(table >= 0, order[table.clamp(min=0).long()], -1)
    state = {"case": case, "bs": bs, "table": table, "lens": _ints(total), "blocks": blocks}
    if case["op"] in ("share", "attend"):
        state["cu"] = torch.arange(len(total) + 1, dtype=torch.int32, device=dev) * case["new"]
        if case["op"] == "share":
            # one to eight drafted tokens; conversations that leave their prompt in its second half
            state["cu"][1:] = torch.randint(1, 9, (len(total),), generator=g, device=dev).cumsum(0)
            common = torch.repeat_interleave(_ints([p // bs for p in prompts]), case["answers"])
            leaves = (common * (0.5 + 0.5 * torch.rand(len(total), generator=g, device=dev))).long()
            col = torch.arange(table.shape[1], device=dev)[None]
            other = blocks + torch.arange(table.numel(), device=dev).reshape(table.shape)
            state["table"] = torch.where((table >= 0) & (col > leaves[:, None]), other.int(), table)
            return state
        # a cache in use: rows of codes and exponents of normal values, drawn from a pool
        pool = torch.randn((4096, D), generator=g, device=dev) * torch.exp(0.3 * torch.randn((4096, 1), generator=g, device=dev))
        c, e = _code(pool, case["dtype"])
        pool_c, pool_s = c[:, 0::2] | c[:, 1::2] << 4, (e + 127).to(torch.uint8)
        pick = torch.randint(0, 4096, (blocks * Hkv * 2 * bs,), generator=g, device=dev, dtype=torch.int32)
        codes = pool_c[pick].reshape(blocks, Hkv, 2, bs, D // 2)
        scales = pool_s[pick].reshape(blocks, Hkv, 2, bs, D // 32)
        T = len(total) * case["new"]
        q = torch.randn((T, case["Hq"], D), generator=g, device=dev).to(_DTYPE[case["dtype"]])[None].transpose(1, 2)
        shared = _share(state)  # the step's plan, which its layers use in turn
        return dict(state, codes=codes, scales=scales, q=q, shared=shared, max_len=max(total))
    # pages of any contents, every layer's in one allocation
    shape = (case["L"], blocks, Hkv, 2, bs)
    state["codes"] = torch.randint(0, 256, (*shape, D // 2), generator=g, device=dev, dtype=torch.uint8)
    state["scales"] = torch.randint(0, 256, (*shape, D // 32), generator=g, device=dev, dtype=torch.uint8)
    # blocks that requests hold are the free list's first, as they were handed out
    state["free"] = order.clone()
    state["used"] = _ints([live])
    if case["op"] == "fork":
        parents, keep = _parents(case, total)
        state.update(parents=_ints(parents), keep=_ints(keep))
    return state


def _code(x, dtype):
    """(codes 0..15, exponents) of float rows x: (..., D), blocks of 32 channels."""
    y = x.reshape(*x.shape[:-1], -1, 32)
    amax = y.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1)
    e = torch.where(amax > 0, e - 3 + (m > 0.875).to(e.dtype), torch.full_like(e, -1000)).clamp(_LOW[dtype], _HIGH[dtype])
    a = torch.ldexp(y.abs(), -e)
    c = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return (c + 8 * (y < 0)).to(torch.uint8).reshape(x.shape), e[..., 0]


def _prepare_verify(case, g):
    dev = _dev()
    counts = _draft_counts(case)
    T, V, dtype = sum(counts) + case["R"], case["V"], _DTYPE[case["dtype"]]
    # a model's probabilities: a few likely tokens and a long tail; the draft's are near them
    logits = 2.5 * torch.randn((T, V), generator=g, device=dev)
    target = torch.softmax(logits, -1)
    logits += 0.7 * torch.randn((T, V), generator=g, device=dev)
    draft = torch.softmax(logits, -1)
    del logits
    # row t of `draft` is what token t was drawn from; the rows' first tokens were not drafted
    cu = torch.zeros(case["R"] + 1, dtype=torch.int32, device=dev)
    cu[1:] = (_ints(counts) + 1).cumsum(0)
    target = torch.cat([target[1:], target[:1]])  # row t of `target` is what follows token t
    race = torch.empty((T, V), device=dev).exponential_(generator=g)
    tokens = (draft.argmax(-1) if case["sure"] else (draft / race).argmax(-1))
    del race
    return {"case": case, "target": target.to(dtype), "draft": None if case["sure"] else draft.to(dtype), "tokens": tokens,
            "cu": cu, "accept": torch.rand((T,), generator=g, device=dev), "sample": torch.rand((case["R"],), generator=g, device=dev),
            "lens": torch.randint(100, 20000, (case["R"],), generator=g, device=dev, dtype=torch.int32) + (cu[1:] - cu[:-1])}


# ---- the plain forms ----

def _share(s):
    """Tokens that each request has in common with its group (skip), and each group's queries as one request's: their first
    tokens (cu) and the keys they see (lens; 0 for every request but a group's first)."""
    table, lens, cu, bs = s["table"], s["lens"].long(), s["cu"].long(), s["bs"]
    R, M = table.shape
    limit = ((lens - (cu[1:] - cu[:-1])).clamp(min=0) // bs).clamp(max=M)
    same = (table[1:] == table[:-1]).long().cumprod(-1).sum(-1)
    common = torch.zeros(R, dtype=torch.long, device=table.device)
    common[1:] = torch.minimum(same, torch.minimum(limit[1:], limit[:-1])) * bs
    first = common < _LEAST
    first[0] = True
    group = first.long().cumsum(0) - 1
    prefix = torch.full((R,), 1 << 40, device=table.device).scatter_reduce_(0, group, torch.where(first, 1 << 40, common), "amin")
    end = torch.zeros(R, dtype=torch.long, device=table.device).scatter_reduce_(
        0, group, torch.arange(1, R + 1, device=table.device), "amax")
    skip = torch.where(prefix[group] < 1 << 40, prefix[group], 0)
    at = torch.where(first, cu[:-1], cu[end[group]])
    return {"skip": skip.int(), "cu": torch.cat([at, cu[-1:]]).int(), "lens": torch.where(first, skip, 0).int()}


def _decode(code, scale):
    """float32 values of codes (0..15) with exponent bytes."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=code.device)
    v = torch.ldexp(grid[(code & 7).long()], scale.to(torch.int32) - 127)
    return torch.where(code >= 8, -v, v)


def _pages(s, L):
    """float32 keys and values (B, Hkv, L, D) of the requests' first L slots, gathered by the block table."""
    case = s["case"]
    D, bs, Hkv = case["D"], s["bs"], case["Hkv"]
    n = -(-L // bs)
    ids = s["table"][:, :n].clamp(min=0).long()
    B, tiles = ids.shape[0], bs // 32
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
    Hq, Hkv, D, N, L = case["Hq"], case["Hkv"], case["D"], case["new"], s["max_len"]
    B, G = s["table"].shape[0], Hq // Hkv
    k, v = _pages(s, L)
    q = s["q"][0].float().reshape(Hkv, G, B, N, D).permute(2, 0, 1, 3, 4).reshape(B, Hkv, G * N, D).contiguous()
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(D))
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    pos = (s["lens"].long() - N)[:, None] + torch.arange(N, device=k.device)  # (B, N)
    seen = torch.arange(L, device=k.device) <= pos[..., None]
    x = torch.where(seen[:, None, None], x.reshape(B, Hkv, G, N, L), -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    norm = x.sum(-1, keepdim=True)
    o = torch.matmul(x.reshape(B, Hkv, G * N, L), v).reshape(B, Hkv, G, N, D) / norm
    return o.permute(0, 3, 1, 2, 4).reshape(B * N, Hq, D).to(s["q"].dtype)[None].transpose(1, 2)


def _ranked(mask, size):
    """Ids of the True entries in ascending order, -1 behind them, ``size`` entries."""
    rank = mask.long().cumsum(0) - 1
    out = torch.full((size + 1,), -1, dtype=torch.long, device=mask.device)
    at = torch.where(mask & (rank < size), rank, size)
    out.scatter_(0, at, torch.arange(mask.numel(), device=mask.device))
    return out[:size]


def _held(table, lens, bs, blocks):
    """(entries of the table that a request of so many tokens holds, -1 elsewhere; the blocks held, as a mask)."""
    col = torch.arange(table.shape[1], device=table.device)[None]
    entry = torch.where((col < (lens[:, None] + bs - 1) // bs) & (table >= 0) & (table < blocks), table.long(), -1)
    mask = torch.zeros(blocks + 1, dtype=torch.bool, device=table.device)
    mask[torch.where(entry >= 0, entry, blocks).reshape(-1)] = True
    return entry, mask[:blocks]


def _fork(s):
    table, bs, blocks, free, codes, scales = s["table"], s["bs"], s["blocks"], s["free"], s["codes"], s["scales"]
    parents, F = s["parents"].long(), s["free"].numel()
    dev = table.device
    lens = torch.minimum(s["lens"][parents], s["keep"]).long().clamp(min=0)
    _, old = _held(table, s["lens"].long(), bs, blocks)
    entry, new = _held(table[parents], lens, bs, blocks)
    R, M = entry.shape
    _, whole = _held(table[parents], lens // bs * bs, bs, blocks)
    # a block that is not full belongs to the first request that will write to it, the others get copies
    col = (lens // bs).clamp(max=M - 1)
    part = torch.where((lens % bs > 0) & (lens // bs < M), entry.gather(1, col[:, None])[:, 0], -1)
    row = torch.arange(R, device=dev)
    first = torch.full((blocks + 1,), R, device=dev).scatter_reduce_(0, torch.where(part >= 0, part, blocks), row, "amin")
    copied = (part >= 0) & (whole[part.clamp(min=0)] | (first[part.clamp(min=0)] != row))
    # blocks that nobody holds any more go back to the list, copies are taken from its top
    used = s["used"][0].long().clamp(0, F)
    given = torch.minimum((old & ~new).sum(), used)
    ids = _ranked(old & ~new, blocks)
    at = torch.arange(F, device=dev) - (used - given)
    free.copy_(torch.where((at >= 0) & (at < given), ids[at.clamp(0, blocks - 1)], free.long()).to(free.dtype))
    k = used - given + copied.long().cumsum(0) - 1
    fresh = torch.where(copied & (k < F), free[k.clamp(0, F - 1)].long(), -1)
    there = torch.arange(M, device=dev)[None] == col[:, None]
    entry = torch.where(there & copied[:, None], fresh[:, None], entry)
    src, dst = part[fresh >= 0], fresh[fresh >= 0]
    codes[:, dst] = codes[:, src]
    scales[:, dst] = scales[:, src]
    return {"table": entry.to(table.dtype), "lens": lens.to(torch.int32), "used": (used - given + copied.sum()).reshape(1).to(torch.int32),
            "free": free, "codes": codes, "scales": scales}


def _compact(s):
    table, bs, blocks, free, codes, scales = s["table"], s["bs"], s["blocks"], s["free"], s["codes"], s["scales"]
    entry, live = _held(table, s["lens"].long(), bs, blocks)
    i = torch.arange(blocks, device=table.device)
    n = live.sum()
    src, dst = _ranked(live & (i >= n), blocks // 2), _ranked(~live & (i < n), blocks // 2)
    src, dst = src[src >= 0], dst[dst >= 0]
    to = i.clone()
    to[src] = dst
    codes[:, dst] = codes[:, src]
    scales[:, dst] = scales[:, src]
    free.copy_(i)
    return {"table": torch.where(entry >= 0, to[entry.clamp(min=0)], -1).to(table.dtype), "used": n.reshape(1).to(torch.int32), "free": free,
            "codes": codes, "scales": scales}


def _verify(s):
    target, draft, tokens, cu = s["target"], s["draft"], s["tokens"], s["cu"].long()
    T, V = target.shape
    dev = target.device
    new = cu[1:] - cu[:-1]
    R = new.numel()
    t = torch.arange(T, device=dev)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    # token t was drafted if another of its request stands before it
    drafted = t > cu[b]
    p = target[(t - 1).clamp(min=0), tokens].double()
    q = torch.ones_like(p) if draft is None else draft[t, tokens].double()
    fails = drafted & ~(s["accept"].double() * q < p)
    stop = torch.where(fails, t - cu[b] - 1, new[b] - 1)
    a = new.scatter_reduce(0, b, stop, "amin")  # tokens accepted
    at = cu[:-1] + a
    x = tokens[(at + 1).clamp(max=T - 1)]
    whole = target[at].double()
    drawn = torch.zeros_like(whole).scatter_(1, x[:, None], 1.0) if draft is None else draft[(at + 1).clamp(max=T - 1)].double()
    w = torch.where((a < new - 1)[:, None], (whole - drawn).clamp(min=0), whole)
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, whole)
    c = w.cumsum(-1)
    nxt = (c <= s["sample"].double()[:, None] * c[:, -1:]).sum(-1)
    last = torch.where(w > 0, torch.arange(V, device=dev), 0).amax(-1)
    nxt = torch.minimum(nxt, last)
    i = t - cu[b]
    follows = torch.where(i < a[b], tokens[(t + 1).clamp(max=T - 1)], torch.where(i == a[b], nxt[b], -1))
    return {"tokens": follows, "accepted": a.int(), "lens": (s["lens"].long() - (new - 1 - a)).int()}


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"share": _share, "attend": _attend, "fork": _fork, "compact": _compact, "verify": _verify}[op](state)
    from gemma_triton_flash_attn_amd import kv4

    s, case = state, state["case"]
    if op == "share":
        return kv4.share(s["table"], s["lens"], s["cu"], block_size=s["bs"])._asdict()
    if op == "attend":
        cache = kv4.Cache(s["codes"], s["scales"], _DTYPE[case["dtype"]])
        return kv4.attention(s["q"], cache, s["table"], s["lens"], s["cu"], max_new=case["new"], softcap=case["softcap"] or None,
                             shared=kv4.Shared(**s["shared"]))
    if op == "verify":
        return kv4.verify(s["target"], s["draft"], s["tokens"], s["accept"], s["sample"], s["lens"], s["cu"])._asdict()
    caches = [kv4.Cache(c, e, _DTYPE[case["dtype"]]) for c, e in zip(s["codes"], s["scales"])]
    if op == "fork":
        f = kv4.fork(caches, s["table"], s["lens"], s["free"], s["used"], parents=s["parents"], keep=s["keep"])
    else:
        f = kv4.compact(caches, s["table"], s["lens"], s["free"])
    return dict(f._asdict(), free=s["free"], codes=s["codes"], scales=s["scales"])


# ---- the definitions ----

def _exact_share(s):
    table, lens, cu = s["table"].tolist(), s["lens"].tolist(), s["cu"].tolist()
    bs, groups = s["bs"], [[0]]
    pairs = [0]
    for b in range(1, len(lens)):
        most = min(max(lens[i] - (cu[i + 1] - cu[i]), 0) // bs for i in (b - 1, b))
        n = 0
        while n < min(most, len(table[b])) and table[b][n] == table[b - 1][n]:
            n += 1
        pairs.append(n * bs)
        if n * bs >= _LEAST:
            groups[-1].append(b)
        else:
            groups.append([b])
    skip, at, seen = [0] * len(lens), [0] * len(lens) + [cu[-1]], [0] * len(lens)
    for g in groups:
        n = min(pairs[b] for b in g[1:]) if len(g) > 1 else 0
        for b in g:
            skip[b], at[b] = n, cu[g[0]] if b == g[0] else cu[g[-1] + 1]
        seen[g[0]] = n
    return {"skip": _ints(skip), "cu": _ints(at), "lens": _ints(seen)}


def _rows(s, side, h, slot):
    """float64 rows of the cache's keys (side 0) or values (side 1) of head h at the slots."""
    D, bs, Hkv = s["case"]["D"], s["bs"], s["case"]["Hkv"]
    t, d = (slot % 32)[:, None], torch.arange(D, device=slot.device)[None]
    page, tile = ((slot // bs) * Hkv + h) * 2 + side, slot % bs // 32
    half, g, r = t // 16, t % 16 // 4, t % 4
    e, block = d - d % 2, d // 32
    if side == 0:
        w = min(D, 128)
        at = e // w * (16 * w) + t * (w // 2) + e % w // 2
        at_s = t * (D // 32) + block % 4 * (D // 128) + block // 4 if D >= 128 else t * 2 + block
    else:
        p, x = e // (D // 16), e % (D // 16)
        at = x // 8 * 2048 + half * 1024 + (g * 16 + p) * 16 + r * 4 + x % 8 // 2 if D >= 128 else (g * 16 + p) * 16 + half * 8 + r * 2 + x // 2
        at_s = (g * (D // 32) + block) * 8 + half * 4 + r
    byte = s["codes"].view(-1)[(page * (bs * D // 2) + tile * (16 * D))[:, None] + at].int()
    power = s["scales"].view(-1)[(page * (bs * D // 32) + tile * D)[:, None] + at_s].double() - 127
    c = torch.where(d % 2 == 1, byte >> 4, byte & 15)
    n = c & 7
    size = torch.where(n < 2, n * 0.5, (1 + 0.5 * (n & 1)) * torch.exp2((n >> 1).double() - 1))
    return torch.where(c > 7, -size, size) * torch.exp2(power)


def _exact_attend(s):
    case = s["case"]
    D, Hq, Hkv, bs, N, cap = case["D"], case["Hq"], case["Hkv"], s["bs"], case["new"], case["softcap"]
    lens, table = s["lens"].tolist(), s["table"].long()
    out = torch.zeros((len(lens) * N, Hq, D), dtype=torch.float64, device=table.device)
    G = Hq // Hkv
    for b, n in enumerate(lens):
        j = torch.arange(n, device=table.device)
        slot = table[b, j // bs] * bs + j % bs
        hidden = (j[None] > torch.arange(n - N, n, device=table.device)[:, None]).repeat(G, 1)
        for h in range(Hkv):
            k, v = _rows(s, 0, h, slot), _rows(s, 1, h, slot)
            q = s["q"][0, h * G:(h + 1) * G, b * N:(b + 1) * N].double().reshape(G * N, D)
            x = q @ k.t().contiguous() / math.sqrt(D)
            x = cap * torch.tanh(x / cap) if cap else x
            o = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v
            out[b * N:(b + 1) * N, h * G:(h + 1) * G] = o.reshape(G, N, D).transpose(0, 1)
    return out[None].transpose(1, 2)


def _exact_fork(s):
    table, lens, bs, blocks = s["table"].tolist(), s["lens"].tolist(), s["bs"], s["blocks"]
    parents, keep, free, used = s["parents"].tolist(), s["keep"].tolist(), s["free"].tolist(), s["used"].item()
    held = {x for row, n in zip(table, lens) for x in row[: -(-n // bs)]}
    n = [min(lens[p], k) for p, k in zip(parents, keep)]
    rows = [table[p][: -(-k // bs)] for p, k in zip(parents, n)]
    whole = {x for row, k in zip(rows, n) for x in row[: k // bs]}
    back = sorted(held - {x for row in rows for x in row})
    for x in reversed(back):
        used -= 1
        free[used] = x
    owner, pairs = {}, []
    for b, (row, k) in enumerate(zip(rows, n)):
        if k % bs:
            x = row[-1]
            if x in whole or owner.setdefault(x, b) != b:
                row[-1] = free[used] if used < len(free) else -1  # the pool is full: `used` tells of it
                pairs += [(x, row[-1])] if used < len(free) else []
                used += 1
    codes, scales = s["codes"], s["scales"]
    for x, y in pairs:
        codes[:, y].copy_(codes[:, x])
        scales[:, y].copy_(scales[:, x])
    M = s["table"].shape[1]
    return {"table": _ints([row + [-1] * (M - len(row)) for row in rows]), "lens": _ints(n), "used": _ints([used]), "free": _ints(free),
            "codes": codes, "scales": scales}


def _exact_compact(s):
    table, lens, bs, blocks = s["table"].tolist(), s["lens"].tolist(), s["bs"], s["blocks"]
    rows = [row[: -(-n // bs)] for row, n in zip(table, lens)]
    live = {x for row in rows for x in row}
    n = len(live)
    to = dict(zip(sorted(x for x in live if x >= n), sorted(set(range(n)) - live)))
    codes, scales = s["codes"], s["scales"]
    for x, y in to.items():
        codes[:, y].copy_(codes[:, x])
        scales[:, y].copy_(scales[:, x])
    M = len(table[0])
    return {"table": _ints([[to.get(x, x) for x in row] + [-1] * (M - len(row)) for row in rows]), "used": _ints([n]),
            "free": _ints(list(range(blocks))), "codes": codes, "scales": scales}


def _exact_verify(s):
    cu, tokens, u, r = s["cu"].tolist(), s["tokens"].tolist(), s["accept"].tolist(), s["sample"].tolist()
    out, accepted = [], []
    for b in range(len(r)):
        t, end = cu[b], cu[b + 1] - 1
        while t < end:
            q = 1.0 if s["draft"] is None else s["draft"][t + 1, tokens[t + 1]].double().item()
            if not u[t + 1] * q < s["target"][t, tokens[t + 1]].double().item():
                break
            out.append(tokens[t + 1])
            t += 1
        w = s["target"][t].double().cpu()
        if t < end:
            z = torch.zeros_like(w)
            z[tokens[t + 1]] = 1.0
            rest = (w - (z if s["draft"] is None else s["draft"][t + 1].double().cpu())).clamp(min=0)
            w = rest if rest.sum() > 0 else w
        c = torch.cumsum(w, 0)
        out.append(int(torch.searchsorted(c, torch.tensor([r[b] * c[-1].item()], dtype=torch.float64), right=True).clamp(max=int(w.nonzero().max()))))
        out += [-1] * (end - t)
        accepted.append(t - cu[b])
    lens = [n - (cu[b + 1] - cu[b] - 1 - accepted[b]) for b, n in enumerate(s["lens"].tolist())]
    return {"tokens": torch.tensor(out, device=s["target"].device), "accepted": _ints(accepted), "lens": _ints(lens)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"share": _exact_share, "attend": _exact_attend, "fork": _exact_fork, "compact": _exact_compact, "verify": _exact_verify}[case["op"]](s)
