"""The operators of the 8-bit key/value cache that their speed is measured on, in their plain form and as calls of ``legion_b200.ops``.

A cache holds e4m3 codes [blocks, kv heads, page, head size] for keys and for values, and for each block and head one scale, a
power of two: a value is its code times the scale of its block. A case names one operator:

  append  new keys and values of every sequence join its blocks. A block's scale is 2^(e - 7) for a largest magnitude in
          [2^e, 2^(e+1)); it only grows, and where it does, the block's older codes are rounded to the new one. Writing a block's
          first cell begins the block anew (its other cells become zero).
  attend  softmax attention of ``new`` query rows per sequence, the last of its ``tokens`` cached ones: one row is a decode
          step, more are a prompt or a part of one. ``weights``: every key's softmax weight, summed over the query heads that
          share its head and over the last ``observe`` rows (0: all), joins a running sum per sequence and head.
  evict   of every sequence and head ``budget`` tokens stay: the first ``first``, the last ``last`` and those with the largest
          sums of weights (equal ones: the earlier), in order, in blocks of their own; codes are rounded to the new blocks' scales,
          the largest of those they come from.

Heads and head sizes are those of the repository's presets (32 / 4 heads of 128, 16 / 2 of 256, 40 / 8 of 128), pages its default.
``ragged``: lengths spread from about half to one and a half times the mean.
"""
from __future__ import annotations

import math

import torch

own = False

HEADS = {"moe": (32, 4, 128), "hybrid": (16, 2, 256), "dense": (40, 8, 128), "small": (4, 2, 64)}
MOST = 3.3895313892515355e38       # largest finite bf16 value: infinities count as this


def listed():
    def case(name, op, model, seqs, tokens, **more):
        return {"name": name, "op": op, "model": model, "seqs": seqs, "tokens": tokens, "page": 64, "new": 1, "ragged": False,
                "window": 0, "softcap": 0.0, "weights": False, "observe": 0, "budget": 0, "first": 0, "last": 0, **more}
    return [
        # a decode step of 16 users writes one token each: the smallest call, all latency
        case("append-16", "append", "moe", 16, 1024),
        # a whole prompt enters the cache
        case("append-8k", "append", "moe", 1, 8192, new=8192),
        # one person chats: every token waits for one short call
        case("decode-1", "attend", "hybrid", 1, 1000),
        # assistants with long histories
        case("decode-16x8k", "attend", "moe", 16, 8192),
        # one question about a book
        case("decode-128k", "attend", "moe", 1, 131072),
        # a report is read before the first answer
        case("prompt-8k", "attend", "moe", 1, 8192, new=8192),
        # questions of mixed lengths admitted in one step
        case("prompts-9", "attend", "hybrid", 9, 611, new=611, ragged=True),
        # the next part of a long document, behind what has been read of it
        case("chunk-32k", "attend", "dense", 1, 33280, new=512),
        # users with chats of all ages whose caches are pruned: each decode step also counts what its tokens looked at
        case("decode-64-weights", "attend", "dense", 64, 1500, ragged=True, weights=True),
        # the end of a prompt says which of its keys matter before the rest is dropped
        case("observe-16k", "attend", "moe", 1, 16384, new=1024, weights=True, observe=64),
        # a chat outgrows its budget
        case("evict-1", "evict", "hybrid", 1, 2500, budget=1024, first=4, last=256),
        # long prompts are cut to an eighth
        case("evict-4x32k", "evict", "moe", 4, 32768, budget=4096, first=4, last=512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "attend", "evict"])
    c = {"op": op, "model": rng.choice(["moe", "hybrid", "dense", "dense", "small"]), "seqs": 1, "tokens": 1, "page": rng.choice([16, 32, 64, 64]),
         "new": 1, "ragged": rng.random() < 0.6, "window": 0, "softcap": 0.0, "weights": False, "observe": 0, "budget": 0, "first": 0, "last": 0}
    if op == "append":
        c["seqs"] = _log(rng, 1, 64)
        c["tokens"] = _log(rng, 64, 65536 // c["seqs"])
        c["new"] = 1 if rng.random() < 0.5 else _log(rng, 2, max(2, min(c["tokens"], 16384 // c["seqs"])))
    elif op == "evict":
        c["seqs"] = _log(rng, 1, 16)
        c["tokens"] = _log(rng, 600, 65536 // c["seqs"])
        c["budget"] = _log(rng, 200, c["tokens"])
        c["first"], c["last"] = rng.choice([0, 1, 4, 16]), rng.randrange(0, c["budget"] // 2)
    else:
        c["window"] = rng.choice([0, 0, 0, 128, 1024])
        c["softcap"] = rng.choice([0.0, 0.0, 0.0, 30.0])
        c["weights"] = rng.random() < 0.3
        if rng.random() < 0.55:
            c["seqs"] = _log(rng, 1, 64)
            c["tokens"] = _log(rng, 64, 131072 // c["seqs"])
        else:
            c["seqs"] = _log(rng, 1, 12)
            c["new"] = _log(rng, 2, 4096 // c["seqs"])
            c["tokens"] = c["new"] + (0 if rng.random() < 0.5 else _log(rng, 64, 4096 // c["seqs"]))
            c["observe"] = rng.choice([0, 32]) if c["weights"] else 0
    return c


def _lengths(case, key="tokens"):
    n, mean = case["seqs"], case[key]
    if not case["ragged"] or n == 1:
        return [mean] * n
    golden = (math.sqrt(5.0) - 1) / 2          # evenly spread, in no order
    return [max(1, int(mean * (0.5 + (i + 1) * golden % 1.0))) for i in range(n)]


def _news(case):
    """New tokens of every sequence: at most its length."""
    if case["new"] == 1:
        return [1] * case["seqs"]
    return [min(a, b) for a, b in zip(_lengths(case, "new"), _lengths(case))]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(7919 * (seed % (1 << 40)) + 17)
    heads, kv, dim = HEADS[case["model"]]
    page, B = case["page"], case["seqs"]
    lens, new = _lengths(case), _news(case)
    width = max(-(-n // page) for n in lens)
    keep = -(-case["budget"] // page)
    n_blocks = sum(-(-n // page) for n in lens) + B * keep + 1
    order = (torch.randperm(n_blocks - 1, device="cuda", generator=g) + 1).tolist()      # block 0 belongs to nobody
    table, dst, at = [], [], 0
    for n in lens:
        k = -(-n // page)
        table.append(order[at:at + k] + [0] * (width - k))
        at += k
    for _ in range(B if keep else 0):
        dst.append(order[at:at + keep])
        at += keep

    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)
    s = {"page": page, "scale": dim ** -0.5, "window": case["window"], "softcap": case["softcap"], "observe": case["observe"],
         "budget": case["budget"], "first": case["first"], "last": case["last"], "max_new": max(new), "max_ctx": max(lens),
         "table": i32(table), "ctx": i32(lens), "cu": i32([sum(new[:i]) for i in range(B + 1)]), "op": case["op"], "sum": None}
    # keys carry a few channels that are far larger than the rest, values a mean of their own; magnitudes differ from block to block
    for name in ("k", "v"):
        x = normal(n_blocks, kv, page, dim)
        x *= torch.exp2(normal(n_blocks, kv, 1, 1) * 0.7)
        if name == "k":
            x *= 1 + 7 * (torch.rand(1, kv, 1, dim, device="cuda", generator=g) < 0.03)
        else:
            x += 0.5 * normal(1, kv, 1, dim)
        scale = _scale_of(x.abs().amax((2, 3)))
        s[name], s[name + "_scale"] = (x / scale[..., None, None]).to(torch.float8_e4m3fn), scale
        del x
    T = sum(new)
    if case["op"] == "attend":
        s["q"] = (normal(T, heads, dim) * 1.5).bfloat16()
        if case["weights"]:
            s["sum"] = torch.rand(B, kv, max(lens), device="cuda", generator=g)
    elif case["op"] == "append":
        s["new_k"], s["new_v"] = normal(T, kv, dim).mul_(2).bfloat16(), normal(T, kv, dim).mul_(2).bfloat16()
        # where the new tokens go, for the plain form
        pos = [(i, p) for i, (n, m) in enumerate(zip(lens, new)) for p in range(n - m, n)]
        s["cell"] = torch.tensor([p % page for _, p in pos], device="cuda")
        s["block"] = torch.tensor([table[i][p // page] for i, p in pos], device="cuda")
        touched = list(dict.fromkeys((i, p // page) for i, p in pos))
        where = {t: j for j, t in enumerate(touched)}
        s["touched"] = torch.tensor([table[i][j] for i, j in touched], device="cuda")
        s["which"] = torch.tensor([where[i, p // page] for i, p in pos], device="cuda")
    else:
        # sums of softmax weights: most keys get next to nothing; equal ones among them
        s["sum"] = torch.round(torch.exp2(normal(B, kv, max(lens)) * 3) * 64) / 64
        s["dst"] = i32(dst)
    return s


def run(s):
    if own:
        from legion_b200 import ops
        cache = ops.Kv8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if s["op"] == "append":
            ops.kv8_append(cache, s["new_k"], s["new_v"], s["table"], s["ctx"], s["cu"], s["max_new"])
            return _cache_of(s)
        if s["op"] == "attend":
            o = ops.kv8_attention(s["q"], cache, s["table"], s["ctx"], s["cu"], s["max_new"], s["scale"], window=s["window"],
                                  softcap=s["softcap"], weights=s["sum"], observe=s["observe"], max_ctx=s["max_ctx"])
            return {"out": o, "sum": s["sum"]}
        lens, kept, w = ops.kv8_evict(cache, s["table"], s["ctx"], s["sum"], s["budget"], s["dst"], keep_first=s["first"],
                                      keep_last=s["last"])
        return {"lens": lens, "kept": kept, "sum": w, **_cache_of(s)}
    return {"append": _append, "attend": _attend, "evict": _evict}[s["op"]](s)


def _cache_of(s):
    return {n: s[n] for n in ("k", "v", "k_scale", "v_scale")}


# ------------------------------------------------------------------------------------------------------ plain form
def _scale_of(amax):
    """2^(e - 7) for magnitudes in [2^e, 2^(e+1)), 2^-60 at least; 0 where there is nothing but zeros."""
    e = torch.frexp(amax).exponent - 1
    power = (((e - 7).clamp_min(-60) + 127) << 23).view(torch.float32)
    return torch.where(amax > 0, power, torch.zeros_like(amax))


def _ratio(a, b):
    return torch.where(b > 0, a / b, torch.zeros_like(b))


def _append(s):
    for name in ("k", "v"):
        x = s["new_" + name].float().clamp(-MOST, MOST)
        codes, scale, touched = s[name], s[name + "_scale"], s["touched"]
        amax = torch.zeros(touched.shape[0], scale.shape[1], device=x.device)
        amax.scatter_reduce_(0, s["which"][:, None].expand(-1, scale.shape[1]), x.abs().nan_to_num(nan=0.0).amax(2), "amax")
        begun = torch.zeros(touched.shape[0], dtype=torch.int32, device=x.device)
        begun.scatter_reduce_(0, s["which"], (s["cell"] == 0).int(), "amax")
        old = torch.where(begun[:, None] > 0, torch.zeros_like(amax), scale[touched])
        now = torch.maximum(old, _scale_of(amax))
        raw = codes.view(torch.uint8)
        older = raw[touched].view(codes.dtype).float() * _ratio(old, now)[..., None, None]
        older = torch.where((begun[:, None] > 0)[..., None, None], torch.zeros_like(older), older)      # NaN too
        raw[touched] = older.to(codes.dtype).view(torch.uint8)
        new = (x * _ratio(torch.ones_like(now), now)[s["which"]][..., None]).clamp(-448, 448).to(codes.dtype)
        raw[s["block"], :, s["cell"]] = new.view(torch.uint8)
        scale[touched] = now
    return _cache_of(s)


def _gathered(s, name):
    """A sequence's keys or values in order, in 32 bits: [seqs, kv heads, width * page, dim]."""
    t = s["table"].long()
    x = s[name].view(torch.uint8)[t].view(s[name].dtype).float() * s[name + "_scale"][t][..., None, None]
    return x.transpose(1, 2).flatten(2, 3)


def _attend(s):
    q, ctx, cu = s["q"], s["ctx"].long(), s["cu"].long()
    k, v = _gathered(s, "k"), _gathered(s, "v")
    B, kv, L, dim = k.shape
    n, group = s["max_new"], q.shape[1] // kv
    new = cu[1:] - cu[:-1]
    row = torch.arange(n, device=q.device)
    used = row < new[:, None]                                                        # [B, n]
    at = torch.where(used, cu[:-1, None] + row, torch.zeros_like(row))
    qs = q[at].float().view(B, n, kv, group, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)      # [B, kv, group * n, dim]
    score = torch.matmul(qs, k.transpose(2, 3)).view(B, kv, group, n, L) * s["scale"]
    if s["softcap"] > 0:
        score = torch.tanh(score / s["softcap"]) * s["softcap"]
    key = torch.arange(L, device=q.device)
    pos = (ctx - new)[:, None] + row
    seen = (key <= pos[..., None]) & used[..., None]                                 # [B, n, L]
    if s["window"] > 0:
        seen &= key > pos[..., None] - s["window"]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    del score
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    v = torch.where((key < ctx[:, None])[:, None, :, None], v, torch.zeros_like(v))
    o = torch.matmul(p.flatten(2, 3), v).view(B, kv, group, n, dim).permute(0, 3, 1, 2, 4).flatten(2, 3)
    out = torch.empty_like(q)
    if s["cu"].shape[0] == 2:
        out.copy_(o[0])
    else:
        flat = torch.where(used, at, torch.full_like(at, q.shape[0])).flatten()      # rows behind a sequence go to a row of their own
        spare = torch.empty(q.shape[0] + 1, *q.shape[1:], dtype=q.dtype, device=q.device)
        spare[flat] = o.flatten(0, 1).to(q.dtype)
        out.copy_(spare[:-1])
    if s["sum"] is not None:
        if s["observe"] > 0:
            p = p * (row >= (new - s["observe"])[:, None])[:, None, None, :, None]
        s["sum"] += p.sum((2, 3))[..., :s["sum"].shape[2]]
    return {"out": out, "sum": s["sum"]}


def _evict(s):
    w, ctx, page, budget = s["sum"], s["ctx"].long(), s["page"], s["budget"]
    B, kv, L = w.shape
    key = torch.arange(L, device=w.device)
    held = (key < ctx[:, None])[:, None]
    always = ((key < s["first"]) | (key >= ctx[:, None] - s["last"]))[:, None]
    rank = torch.where(held, torch.where(always, torch.full_like(w, math.inf), w), torch.full_like(w, -math.inf))
    best = torch.sort(rank, dim=2, descending=True, stable=True).indices[..., :budget]
    best = torch.sort(torch.where(best < ctx[:, None, None], best, torch.full_like(best, 1 << 40)), dim=2).values
    short = budget - best.shape[2]
    if short > 0:
        best = torch.nn.functional.pad(best, (0, short), value=1 << 40)
    stays = best < (1 << 40)
    idx = torch.where(stays, best, torch.zeros_like(best))
    h = torch.arange(kv, device=w.device)[None, :, None]
    b = torch.arange(B, device=w.device)[:, None, None]
    src = s["table"].long()[b, idx // page]                                          # [B, kv, budget]
    blocks = -(-budget // page)
    pad = blocks * page - budget
    dst = s["dst"].long()[:, :blocks]
    written = (torch.arange(blocks, device=w.device) * page < ctx.clamp_max(budget)[:, None])     # [B, blocks]
    for name in ("k", "v"):
        codes, scale = s[name], s[name + "_scale"]
        raw = codes.view(torch.uint8)
        from_scale = torch.where(stays, scale[src, h], torch.zeros_like(w[:, :1, :1]))
        from_scale = torch.nn.functional.pad(from_scale, (0, pad)).view(B, kv, blocks, page)
        now = from_scale.amax(3)                                                     # [B, kv, blocks]
        x = raw[src, h, idx % page].view(codes.dtype).float()
        x = torch.where(stays[..., None], x, torch.zeros_like(x))
        x = torch.nn.functional.pad(x, (0, 0, 0, pad)).view(B, kv, blocks, page, -1) * _ratio(from_scale, now[..., None])[..., None]
        x = x.to(codes.dtype).view(torch.uint8).transpose(1, 2)
        raw[dst] = torch.where(written[..., None, None, None], x, raw[dst])
        scale[dst] = torch.where(written[..., None], now.transpose(1, 2), scale[dst])
    return {"lens": ctx.clamp_max(budget).int(), "kept": torch.where(stays, best, torch.full_like(best, -1)).int(),
            "sum": torch.where(stays, torch.gather(w, 2, idx), torch.zeros_like(w[:, :1, :1])), **_cache_of(s)}


# ---------------------------------------------------------------------------------------------------- what it costs
def work(case):
    heads, kv, dim = HEADS[case["model"]]
    lens, new = _lengths(case), _news(case)
    page = case["page"]
    if case["op"] == "append":
        # bf16 rows in, codes out, and the scales of the blocks that they fall in
        blocks = sum(-(-n // page) - (n - m) // page for n, m in zip(lens, new))
        return {"bytes": 2 * kv * (sum(new) * dim * 3 + blocks * 8), "flops": 2 * kv * sum(new) * dim * 2}
    if case["op"] == "evict":
        stay = [min(n, case["budget"]) for n in lens]
        rows = sum(stay) * kv
        return {"bytes": sum(lens) * kv * 4 + rows * (2 * 2 * dim + 8) + 2 * 2 * 4 * -(-rows // page), "flops": rows * 2 * dim}
    w = case["window"]
    keys, pairs, looked = 0, 0, 0
    for n, m in zip(lens, new):
        span = n if w == 0 else min(n, w + m - 1)
        keys += span
        see = [min(p, w) if w else p for p in range(n - m + 1, n + 1)]
        pairs += sum(see)
        looked += sum(see[-case["observe"]:] if case["observe"] else see)
    bytes_ = keys * kv * 2 * (dim + 4 / page) + sum(new) * heads * dim * 4
    flops = 4 * pairs * heads * dim
    if case["weights"]:
        bytes_ += 8 * kv * keys
        flops += 2 * looked * heads
        if case["observe"]:
            flops += 2 * looked * heads * dim          # these rows' scores once more, when their sums are known
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def _two(e):
    """2^e of whole numbers."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _e4m3(x):
    """float64 values rounded to e4m3 (ties to even, magnitudes to 448)."""
    mag = x.abs().clamp(max=448.0)
    step = _two(torch.floor(torch.log2(mag.clamp(min=2.0 ** -6)) + 1e-12) - 3)      # (codes lie further apart than that)
    return torch.copysign((torch.round(mag / step) * step).clamp(max=448.0), x)


def _power(amax):
    """The block scale of a largest magnitude."""
    e = torch.floor(torch.log2(amax.clamp(min=1e-300)))
    e = torch.where(_two(e) > amax, e - 1, e)
    e = torch.where(_two(e + 1) <= amax, e + 1, e)
    return torch.where(amax > 0, _two((e - 7).clamp(min=-60.0)), torch.zeros_like(amax))


def exact(case, seed):
    s = prepare(case, seed)
    lens, new = _lengths(case), _news(case)
    page, table, first = case["page"], s["table"].tolist(), s["cu"].tolist()
    if case["op"] == "append":
        r = {n: s[n].double() for n in ("k", "v", "k_scale", "v_scale")}
        for name in ("k", "v"):
            c, sc, x = r[name], r[name + "_scale"], s["new_" + name].double()
            for i, (n, m) in enumerate(zip(lens, new)):
                p = n - m
                while p < n:
                    end = min(n, (p // page + 1) * page)
                    blk, rows = table[i][p // page], x[first[i] + p - (n - m):first[i] + end - (n - m)].transpose(0, 1)
                    need = _power(rows.abs().amax((1, 2)))
                    if p % page == 0:
                        c[blk], sc[blk] = 0, 0
                    now = torch.maximum(need, sc[blk])
                    by = torch.where(now > 0, now, torch.ones_like(now))[:, None, None]
                    c[blk] = _e4m3(c[blk] * sc[blk][:, None, None] / by)
                    c[blk, :, p % page:p % page + end - p] = _e4m3(rows / by)
                    sc[blk] = now
                    p = end
        return r
    if case["op"] == "evict":
        r = {n: s[n].double() for n in ("k", "v", "k_scale", "v_scale")}
        B, kv = s["sum"].shape[:2]
        out = torch.zeros(B, kv, case["budget"], dtype=torch.float64, device="cuda")
        for i, n in enumerate(lens):
            blocks = s["table"][i].long()
            for h in range(kv):
                w = s["sum"][i, h, :n].double()
                w[:case["first"]] = math.inf
                w[max(0, n - case["last"]):] = math.inf
                kept = torch.argsort(-w, stable=True)[:case["budget"]].sort().values
                m = kept.numel()
                out[i, h, :m] = s["sum"][i, h].double()[kept]
                for name in ("k", "v"):
                    sc = s[name + "_scale"].double()[blocks[kept // page], h]
                    val = s[name].view(torch.uint8)[blocks[kept // page], h, kept % page].view(s[name].dtype).double() * sc[:, None]
                    for j in range(0, m, page):
                        blk = int(s["dst"][i, j // page])
                        now = sc[j:j + page].max()
                        r[name][blk, h] = 0
                        if now > 0:
                            r[name][blk, h, :min(page, m - j)] = _e4m3(val[j:j + page] / now)
                        r[name + "_scale"][blk, h] = now
        return {"lens": None, "kept": None, "sum": out, **r}
    q = s["q"].double()
    group = q.shape[1] // s["k"].shape[1]
    out = torch.zeros_like(q)
    total = None if s["sum"] is None else s["sum"].double()
    for i, (n, m) in enumerate(zip(lens, new)):
        blocks = s["table"][i, :-(-n // page)].long()
        key, row = torch.arange(n, device="cuda"), torch.arange(n - m, n, device="cuda")[:, None]
        hidden = key > row
        if case["window"]:
            hidden |= key <= row - case["window"]
        for h in range(s["k"].shape[1]):
            k, v = ((s[x].view(torch.uint8)[blocks, h].view(s[x].dtype).double()
                     * s[x + "_scale"].double()[blocks, h][:, None, None]).flatten(0, 1)[:n] for x in ("k", "v"))
            for j in range(h * group, (h + 1) * group):
                a = (q[first[i]:first[i + 1], j] @ k.T) * s["scale"]
                if case["softcap"]:
                    a = case["softcap"] * torch.tanh(a / case["softcap"])
                p = torch.softmax(a.masked_fill_(hidden, -math.inf), dim=1)
                out[first[i]:first[i + 1], j] = p @ v
                if total is not None:
                    total[i, h, :n] += (p[-case["observe"]:] if case["observe"] else p).sum(0)
    return {"out": out, "sum": total}
