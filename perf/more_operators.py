"""A serving step's dense attention as cases that can be timed and checked: the step's block table and slot maps built on
the GPU, the attention of whole prompts before anything of them is cached, and the attention of new tokens (one each, or a
chunk) over every cached latent row of their request.

    own                  whether run() calls this package's operators or their plain forms in torch
    listed()             the cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  the queries, caches, tables and buffers that a serving program holds before the call
    run(state)           one call (maps: a step and the trim that takes it back) and its outputs
    work(case)           bytes and operations that the call cannot do without
    exact(case, seed)    the outputs in 64 bits
"""
import math
import random

import torch

own = False

DEV = "cuda"
LAT, ROPE = 512, 64                # latent and rotary widths of a cache row
QK = LAT + ROPE
GROUP = 128                        # latent values per scale of a 656-byte row
KV_SCALE = 0.25                    # per-tensor scale of the fp8 (576-byte) cache
SM = 192 ** -0.5                   # softmax scale of the 128 + 64 wide heads
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
PAIRS = 1 << 31                    # scores of a case, at most (the plain forms hold them in 32 bits)


# ---------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one user's token enters a step
        dict(name="maps_1", kind="maps", requests=1, tokens=1, ctx=4000, block=64, padded=0, spread=0),
        # a decode batch with a few drafted tokens each, padded to a captured graph's size
        dict(name="maps_decode", kind="maps", requests=256, tokens=740, ctx=20000, block=64, padded=28, spread=1),
        # prompts of many users enter at once
        dict(name="maps_prefill", kind="maps", requests=48, tokens=32768, ctx=0, block=16, padded=0, spread=3),
        # one short prompt, expanded heads of 128 + 64 against values of 128
        dict(name="prompt_short", kind="prompt", requests=1, tokens=77, heads=128, kv_heads=128, dim=192, vdim=128,
             causal=True, dtype="bf16", spread=0),
        # prompts of many lengths in one batch, four query heads to a key head
        dict(name="prompt_ragged", kind="prompt", requests=17, tokens=8003, heads=32, kv_heads=8, dim=128, vdim=128,
             causal=True, dtype="bf16", spread=3),
        # prompts without a mask (an encoder's), half precision, narrow heads
        dict(name="prompt_full", kind="prompt", requests=4, tokens=8192, heads=16, kv_heads=16, dim=64, vdim=64,
             causal=False, dtype="fp16", spread=0),
        # a long prompt, expanded heads
        dict(name="prompt_long", kind="prompt", requests=1, tokens=4096, heads=128, kv_heads=128, dim=192, vdim=128,
             causal=True, dtype="bf16", spread=0),
        # one user's token far into a long context
        dict(name="chunk_1", kind="chunk", requests=1, tokens=1, heads=128, ctx=65536, row=656, block=64, spread=0),
        # a full decode batch, contexts of many lengths
        dict(name="chunk_decode_64", kind="chunk", requests=64, tokens=64, heads=128, ctx=6000, row=656, block=64, spread=2),
        # a tensor-parallel rank (16 of 128 heads), per-tensor fp8 cache, long contexts
        dict(name="chunk_decode_tp8", kind="chunk", requests=48, tokens=48, heads=16, ctx=20000, row=576, block=64, spread=2),
        # decoding tokens beside chunks of two prompts, 32 heads a rank, small pages
        dict(name="chunk_mixed", kind="chunk", requests=10, tokens=1009, heads=32, ctx=3001, row=656, block=16, spread=4),
        # a prefill chunk of one long request
        dict(name="chunk_prefill", kind="chunk", requests=1, tokens=1024, heads=128, ctx=16384, row=576, block=64, spread=0),
    ]


def _logu(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["maps", "prompt", "prompt", "chunk", "chunk", "chunk"])
    if kind == "maps":
        B = _logu(rng, 1, 1024)
        tokens = _logu(rng, B, max(B, 32768)) if rng.random() < 0.5 else B * rng.choice([1, 1, 3])
        return dict(kind="maps", requests=B, tokens=tokens, ctx=_logu(rng, 1, 40000), block=rng.choice([16, 64, 64, 48]),
                    padded=rng.choice([0, 0, 37]), spread=rng.choice([0, 1, 3]))
    if kind == "prompt":
        dim, vdim = rng.choice([(192, 128), (192, 128), (128, 128), (64, 64), (256, 256), (96, 96), (72, 40)])
        kv = rng.choice([1, 2, 8, 16])
        heads = kv * rng.choice([1, 1, 4, 5, 8])
        B = _logu(rng, 1, 32)
        tokens = max(B, _logu(rng, 1, 8192))
        while _padded_pairs(dict(kind="prompt", requests=B, tokens=tokens, heads=heads, spread=3)) > PAIRS:
            tokens = max(B, tokens // 2)
        return dict(kind="prompt", requests=B, tokens=tokens, heads=heads, kv_heads=kv, dim=dim, vdim=vdim,
                    causal=rng.random() < 0.8, dtype=rng.choice(["bf16", "bf16", "fp16"]), spread=rng.choice([0, 1, 3]))
    decode = rng.random() < 0.5
    B = _logu(rng, 1, 96)
    tokens = B * rng.choice([1, 1, 2, 4]) if decode else max(B, _logu(rng, 1, 1024))
    c = dict(kind="chunk", requests=B, tokens=tokens, heads=rng.choice([128, 64, 32, 16, 8, 40]), ctx=_logu(rng, 1, 65536),
             row=rng.choice([656, 576]), block=rng.choice([64, 64, 16, 128, 48]), spread=rng.choice([0, 2, 2]) if decode else 4)
    while _padded_pairs(c) > PAIRS or B * c["ctx"] > 1 << 20:
        c["ctx"] = max(1, c["ctx"] // 2)
        if c["ctx"] < 256 and c["tokens"] > B:
            c["tokens"] = max(B, c["tokens"] // 2)
    return c


def _lens(case):
    """New tokens of each request. spread 0: as even as they go; 1: one token at least, the others anywhere; 3: lengths
    that differ tenfold and more; 4: one token each but for two requests that share the rest."""
    B, n, kind = case["requests"], case["tokens"], case["spread"]
    rng = random.Random(7919 * B + n)
    if kind in (0, 2):
        return [n // B + (i < n % B) for i in range(B)]
    if kind == 4 and B > 2:
        lens = [1] * B
        lens[B // 2] += (n - B) // 3
        lens[B // 3] += n - B - (n - B) // 3
        return lens
    lens, rest = [1] * B, n - B
    weight = [rng.random() ** kind for _ in range(B)]
    total = sum(weight)
    for i in range(B):
        lens[i] += int(rest * weight[i] / total)
    lens[B // 2] += n - sum(lens)
    return lens


def _contexts(case):
    """Rows of each request that are cached before the step."""
    B, ctx = case["requests"], case["ctx"]
    if case["spread"] == 0:
        return [ctx] * B
    rng = random.Random(104729 * B + ctx)
    return [ctx // 5 + rng.randrange(ctx - ctx // 5 + 1) for _ in range(B)]


def _seqs(case):
    """Cached rows of each request with its new ones: the new tokens are the last of them (chunk: ctx counts them)."""
    return [max(c, n) for c, n in zip(_contexts(case), _lens(case))]


def _padded_pairs(case):
    lens = _lens(case)
    longest = max(_seqs(case)) if case["kind"] == "chunk" else max(lens)
    return case["requests"] * max(lens) * case["heads"] * longest


# ---------------------------------------------------------------------------------------------- inputs from the seed
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return _ints(at)


def _blocks(n, block):
    return -(-n // block)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=case)
    (_prepare_maps if case["kind"] == "maps" else _prepare_prompt if case["kind"] == "prompt" else _prepare_chunk)(case, g, s)
    return s


def _prepare_maps(case, g, s):
    """A pool in use: requests that hold the pages of their cached rows, the rest free in no order."""
    B, bs, lens, ctx = case["requests"], case["block"], _lens(case), _contexts(case)
    held = [_blocks(c, bs) for c in ctx]
    width = max(_blocks(c + n, bs) for c, n in zip(ctx, lens)) + 3
    spare = sum(_blocks(c + n, bs) - h for c, n, h in zip(ctx, lens, held)) + 100
    pages = torch.randperm(sum(held) + spare, generator=g, device=DEV).to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    table[torch.arange(width, device=DEV) < _ints(held)[:, None]] = pages[:sum(held)]
    free = torch.full((pages.shape[0],), -1, dtype=torch.int32, device=DEV)
    free[:spare] = pages[sum(held):]
    n = case["tokens"] + case["padded"]
    s.update(table=table, lens=_ints(ctx), held=_ints(held), free=free, state=_ints([spare, 0, 0, 0]), n=n, block=bs,
             new=_ints(lens), keep=_ints(ctx), start=torch.empty(B + 1, dtype=torch.int32, device=DEV),
             req=torch.empty(n, dtype=torch.int32, device=DEV), positions=torch.empty(n, dtype=torch.int64, device=DEV),
             slots=torch.empty(n, dtype=torch.int64, device=DEV))


def _prepare_prompt(case, g, s):
    T, H, Hk, D, Dv, dt = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "vdim", "dtype"))
    lens = _lens(case)
    # keys share a direction that some queries seek: rows of scores with peaks as well as flat ones
    common = _randn(g, Hk, D)
    s["k"] = (_randn(g, T, Hk, D) + 0.5 * common).to(TYPES[dt])
    s["q"] = (_randn(g, T, H, D) + _randn(g, T, H, 1) * 0.3 * common.repeat_interleave(H // Hk, 0)).to(TYPES[dt])
    s["v"] = _randn(g, T, Hk, Dv).to(TYPES[dt])
    s["start"], s["longest"], s["scale"] = _starts(lens), max(lens), D ** -0.5
    s["out"] = torch.empty(T, H, Dv, dtype=TYPES[dt], device=DEV)
    s["lse"] = torch.empty(T, H, dtype=torch.float32, device=DEV)


def _prepare_chunk(case, g, s):
    T, H, row, bs = case["tokens"], case["heads"], case["row"], case["block"]
    lens, seqs = _lens(case), _seqs(case)
    held = [_blocks(n, bs) for n in seqs]
    width = max(held) + 1
    pages = sum(held) + 5
    cache = torch.empty(pages, bs, row, dtype=torch.uint8, device=DEV)
    for at in range(0, pages, 4096):                            # 4096 pages at a time
        part = cache[at:at + 4096].view(-1, row)
        n = part.shape[0]
        if row == 576:
            part.copy_((_randn(g, n, QK) / KV_SCALE).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
        else:
            lat = _randn(g, n, LAT // GROUP, GROUP) * torch.exp(0.3 * _randn(g, n, LAT // GROUP, 1))
            sc = lat.abs().amax(2, keepdim=True) / 448.0
            part[:, :LAT] = (lat / sc).to(torch.float8_e4m3fn).view(torch.uint8).view(n, LAT)
            part[:, LAT:LAT + 16] = sc.view(n, LAT // GROUP).view(torch.uint8)
            part[:, LAT + 16:] = _randn(g, n, ROPE).to(torch.bfloat16).view(torch.uint8)
    table = torch.full((case["requests"], width), -1, dtype=torch.int32, device=DEV)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    has = torch.arange(width, device=DEV) < _ints(held)[:, None]
    table[has] = order[:sum(held)]
    # what earlier requests left behind each sequence's end, values that are no numbers among it
    for b, n in enumerate(seqs):
        if n % bs:
            cache[table[b, n // bs].long(), n % bs:] = 0x7F
    s["q"] = _randn(g, T, H, QK).to(torch.bfloat16)
    s.update(cache=cache, table=table, seqs=_ints(seqs), start=_starts(lens), longest=max(seqs), widest=max(lens),
             out=torch.empty(T, H, LAT, dtype=torch.bfloat16, device=DEV),
             lse=torch.empty(T, H, dtype=torch.float32, device=DEV))


# ---------------------------------------------------------------------------------------------- one call
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from arcagi2_flashnext_dots3_amd import kernels, paging
    c = s["case"]
    if c["kind"] == "maps":
        if "pool" not in s:
            s["pool"] = paging.PagePool.over(s["table"], s["lens"], s["held"], s["free"], s["state"], s["block"])
        kernels.page_step(s["pool"], s["new"], s["n"], start=s["start"], req=s["req"], positions=s["positions"],
                          slots=s["slots"])
        kernels.page_trim(s["pool"], s["keep"])
        return _maps(s)
    if c["kind"] == "prompt":
        kernels.attend_prompt(s["q"], s["k"], s["v"], s["start"], s["scale"], causal=c["causal"], out=s["out"], lse=s["lse"])
    else:
        kernels.attend_chunk(s["q"], s["cache"], s["table"], s["seqs"], s["start"], SM,
                             KV_SCALE if c["row"] == 576 else 1.0, max_seq_len=s["longest"], out=s["out"], lse=s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def _maps(s):
    got = {k: s[k] for k in ("start", "req", "positions", "slots", "table", "lens", "held", "free")}
    return {**got, "count": s["state"][:2]}


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "maps":
        _step_plain(s)
        _trim_plain(s)
        return _maps(s)
    return (_prompt_plain if kind == "prompt" else _chunk_plain)(s)


def _step_plain(s):
    bs, n, width, last = s["block"], s["n"], s["table"].shape[1], s["new"].shape[0] - 1
    new = s["new"].clamp(min=0)
    s["start"][0] = 0
    s["start"][1:] = new.cumsum(0)
    need = ((((s["lens"] + new + bs - 1) // bs).clamp(max=width)) - s["held"]).clamp(min=0)
    off = need.cumsum(0) - need
    count = s["state"][0]
    got = torch.minimum(need, (count - off).clamp(min=0))
    col = torch.arange(width, device=DEV, dtype=torch.int32) - s["held"][:, None]
    take = (col >= 0) & (col < got[:, None])
    page = s["free"][(count - 1 - off[:, None] - col).clamp(min=0, max=s["free"].shape[0] - 1).long()]
    s["table"].copy_(torch.where(take, page, s["table"]))
    at = torch.arange(n, device=DEV, dtype=torch.int32)
    in_step = at < s["start"][-1]
    req = torch.searchsorted(s["start"][1:], at, right=True).clamp(max=last)
    pos = s["lens"][req] + at - s["start"][req]
    has = in_step & (pos // bs < (s["held"] + got)[req])
    page = s["table"][req, (pos // bs).clamp(max=width - 1).long()].long()
    s["req"].copy_(torch.where(in_step, req, last))
    s["positions"].copy_(torch.where(in_step, pos, 0))
    s["slots"].copy_(torch.where(has, page * bs + pos % bs, -1))
    s["lens"] += new
    s["held"] += got
    s["state"][0] -= got.sum()
    s["state"][1] = (need - got).sum()


def _trim_plain(s):
    bs, width = s["block"], s["table"].shape[1]
    s["lens"].copy_(torch.minimum(s["lens"], s["keep"].clamp(min=0)))
    left = torch.minimum(s["held"], (s["lens"] + bs - 1) // bs)
    back = s["held"] - left
    off = back.cumsum(0) - back
    col = torch.arange(width, device=DEV, dtype=torch.int32)
    out = (col >= left[:, None]) & (col < s["held"][:, None])
    size = s["free"].shape[0]
    to = s["state"][0] + back.sum() - 1 - off[:, None] - (col - left[:, None])
    room = torch.nn.functional.pad(s["free"], (0, 1))
    room[torch.where(out, to, size).long()] = s["table"]       # (entries that stay go behind the end)
    s["free"].copy_(room[:size])
    s["table"].masked_fill_(out, -1)
    s["state"][0] += back.sum()
    s["held"].copy_(left)


def _pad(x, start, longest):
    """Tokens [T, ...] as [requests, longest, ...] in 32 bits (rows behind a sequence's end: others', to be masked)."""
    at = start[:-1, None].long() + torch.arange(longest, device=DEV)
    return x[at.clamp(max=x.shape[0] - 1)].float()


def _attended(scores, seen, values):
    """Masked softmax over the last axis in 32 bits, its product with the values, and the log of its sum."""
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    return (p @ values) / total, (top + total.log())[..., 0]


def _prompt_plain(s):
    c, start, N = s["case"], s["start"], s["longest"]
    T, H, Hk = c["tokens"], c["heads"], c["kv_heads"]
    q, k, v = (_pad(s[x], start, N).transpose(1, 2) for x in "qkv")               # [B, heads, N, D]
    k, v = (x.repeat_interleave(H // Hk, 1).contiguous() for x in (k, v))
    i = torch.arange(N, device=DEV)
    lens = (start[1:] - start[:-1]).long()
    seen = (i < lens[:, None])[:, None, None, :]
    if c["causal"]:
        seen = seen & (i[None, :] <= i[:, None])
    o, lse = _attended((q.contiguous() @ k.transpose(2, 3)).mul_(s["scale"]), seen, v)
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(start[1:].long(), t, right=True)
    at = t - start.long()[b]
    s["out"].copy_(o[b, :, at])
    s["lse"].copy_(lse[b, :, at])
    return {"out": s["out"], "lse": s["lse"]}


def _rows(raw):
    """Cache rows of bytes [..., row] as 576 values in 32 bits."""
    if raw.shape[-1] == QK:
        return raw.view(torch.float8_e4m3fn).float() * KV_SCALE
    sc = raw[..., LAT:LAT + 16].contiguous().view(torch.float32)
    lat = raw[..., :LAT].contiguous().view(torch.float8_e4m3fn).float() * sc.repeat_interleave(GROUP, -1)
    return torch.cat((lat, raw[..., LAT + 16:].contiguous().view(torch.bfloat16).float()), -1)


def _chunk_plain(s):
    c, start, N, L = s["case"], s["start"], s["widest"], s["longest"]
    T, H, bs, B = c["tokens"], c["heads"], c["block"], c["requests"]
    lens, seqs = (start[1:] - start[:-1]).long(), s["seqs"].long()
    p = torch.arange(L, device=DEV)
    page = s["table"][:, p // bs].long()                                            # [B, L]
    live = (p < seqs[:, None]) & (page >= 0)
    rows = _rows(s["cache"][page.clamp(min=0), p % bs]).masked_fill_(~live[..., None], 0.0)
    q = _pad(s["q"], start, N)                                                      # [B, N, H, 576]
    limit = (seqs - lens)[:, None] + torch.arange(N, device=DEV) + 1                # [B, N]
    seen = (live[:, None] & (p < limit[..., None]))[:, :, None]
    scores = (q.view(B, N * H, QK) @ rows.transpose(1, 2)).mul_(SM).view(B, N, H, L)
    o, lse = _attended(scores, seen, rows[:, None, :, :LAT].contiguous())
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(start[1:].long(), t, right=True)
    at = t - start.long()[b]
    s["out"].copy_(o[b, at])
    s["lse"].copy_(lse[b, at])
    return {"out": s["out"], "lse": s["lse"]}


# ---------------------------------------------------------------------------------------------- what it cannot do without
def work(case):
    lens = _lens(case)
    T, kind = case["tokens"], case["kind"]
    if kind == "maps":
        bs, n, ctx = case["block"], T + case["padded"], _contexts(case)
        fresh = sum(_blocks(c + m, bs) - _blocks(c, bs) for c, m in zip(ctx, lens))
        # a step: lengths and pages held read and written, maps written, new pages taken and entered; a trim: back again
        return {"bytes": 20 * n + 4 * (len(lens) + 1) + 32 * len(lens) + 16 * fresh, "flops": n}
    H = case["heads"]
    if kind == "prompt":
        Hk, D, Dv = case["kv_heads"], case["dim"], case["vdim"]
        pairs = sum(m * (m + 1) // 2 if case["causal"] else m * m for m in lens)
        return {"bytes": 2 * T * (H * D + Hk * D + Hk * Dv + H * Dv) + 4 * T * H, "flops": 2 * pairs * H * (D + Dv)}
    seqs = _seqs(case)
    pairs = sum(m * (n - m) + m * (m + 1) // 2 for m, n in zip(lens, seqs))
    entries = sum(_blocks(n, case["block"]) for n in seqs)
    return {"bytes": sum(seqs) * case["row"] + 4 * entries + 2 * T * H * (QK + LAT) + 4 * T * H,
            "flops": 2 * pairs * H * (QK + LAT)}


# ---------------------------------------------------------------------------------------------- the outputs in 64 bits
def _softmax64(q, k, v, seen):
    """q [h, n, D], k [h or 1, L, D], v [h or 1, L, Dv], all float64; seen [n, L]."""
    z = torch.matmul(q, k.transpose(1, 2).contiguous())
    z = torch.where(seen, z, -math.inf)
    lse = torch.logsumexp(z, 2)
    return torch.matmul(torch.exp(z - lse[..., None]), v), lse


def exact(case, seed):
    kind = case["kind"]
    if kind == "maps":
        return None
    s = prepare(case, seed)
    lens, H, T = _lens(case), case["heads"], case["tokens"]
    out = torch.empty(T, H, s["out"].shape[2], dtype=torch.float64, device=DEV)
    lse = torch.empty(T, H, dtype=torch.float64, device=DEV)
    t0 = 0
    for b, n in enumerate(lens):
        q = s["q"][t0:t0 + n].double()
        if kind == "prompt":
            L, group = n, H // case["kv_heads"]
            seen = torch.ones(n, L, dtype=torch.bool, device=DEV)
            if case["causal"]:
                seen = seen.tril()
        else:
            L = int(s["seqs"][b])
            at = torch.arange(L, device=DEV)
            raw = s["cache"][s["table"][b].long()[at // case["block"]], at % case["block"]]
            k = _rows64(raw)
            seen = at <= (L - n + torch.arange(n, device=DEV))[:, None]
        step = max(1, min(H, (1 << 27) // (n * L)))              # heads at a time
        for h in range(0, H, step):
            qh = q[:, h:h + step].transpose(0, 1)
            if kind == "prompt":
                at = torch.arange(h, min(h + step, H), device=DEV) // group
                kh, vh = (s[x][t0:t0 + n].double().transpose(0, 1)[at].contiguous() for x in "kv")
                o, z = _softmax64(qh.contiguous() * s["scale"], kh, vh, seen)
            else:
                m = qh.shape[0]
                o, z = _softmax64(qh.reshape(1, m * n, QK) * SM, k[None], k[None, :, :LAT].contiguous(), seen.repeat(m, 1))
                o, z = o.view(m, n, LAT), z.view(m, n)
            out[t0:t0 + n, h:h + step] = o.transpose(0, 1)
            lse[t0:t0 + n, h:h + step] = z.transpose(0, 1)
        t0 += n
    return {"out": out, "lse": lse}


def _rows64(raw):
    n = raw.shape[0]
    if raw.shape[1] == QK:
        return raw.view(torch.float8_e4m3fn).double() * KV_SCALE
    k = torch.empty(n, QK, dtype=torch.float64, device=DEV)
    codes = raw[:, :LAT].contiguous().view(torch.float8_e4m3fn).double().view(n, LAT // GROUP, GROUP)
    k[:, :LAT] = (codes * raw[:, LAT:LAT + 16].contiguous().view(torch.float32).double()[..., None]).view(n, LAT)
    k[:, LAT:] = raw[:, LAT + 16:].contiguous().view(torch.bfloat16).double()
    return k
