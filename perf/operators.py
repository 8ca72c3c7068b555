"""The serving operators that are measured, in their plain form and as calls of the framework.

A cache held in 4 bits lies in pages of `page` tokens.  One page of one layer is `heads` x `page / 32` tiles;
a tile holds 32 tokens of one head: the keys' codes (a row of d/2 bytes a token, two dimensions a byte, the
lower one in the low bits), the keys' 32 scales (f32), the values' codes, the values' 32 scales.  The values'
codes are rows of d/4 16-bit granules in which the tokens 2p and 2p+1 alternate.  A code n stands for
n - 7.5, times its row's scale, in a rotated basis: y = R x, R = product over rounds of H diag(signs) / sqrt(d).

Kinds of cases: `attend` (attention over the cache), `append` (rows into the cache and back out of it),
`pages` (extending, forking, copying, compacting, freeing) and `prompt` (attention over whole packed prompts).
"""
import math
import random

import torch

own = False
DEV = "cuda" if torch.cuda.is_available() else "cpu"
TILE = 32
STEP = 0.3352  # of a row's standard deviation: the step of the best uniform 16-level quantiser of a Gaussian


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one user's short chat, one token: the smallest call, all latency
        dict(name="attend-1x300", kind="attend", seqs=1, lo=300, hi=300, q=1, hq=8, heads=2, d=64, page=64, rounds=1, type="float16"),
        # an ordinary decode batch of grouped-head attention, lengths as users have them
        dict(name="attend-16x8k", kind="attend", seqs=16, lo=700, hi=8001, q=1, hq=32, heads=8, d=128, page=64, rounds=1, type="bfloat16"),
        # the largest decode batch: many users with long contexts
        dict(name="attend-64x20k", kind="attend", seqs=64, lo=1000, hi=20000, q=1, hq=64, heads=8, d=128, page=64, rounds=1, type="bfloat16"),
        # checking drafted tokens, up to five a sequence, every head its own keys
        dict(name="attend-verify", kind="attend", seqs=8, lo=33, hi=4500, q=5, hq=16, heads=16, d=128, page=32, rounds=1, type="float16"),
        # a decode step's new rows into the cache, and back
        dict(name="append-64x1", kind="append", seqs=64, lo=50, hi=6000, q=1, hq=8, heads=8, d=128, page=64, rounds=1, type="bfloat16"),
        # whole prompts' rows into the cache, and back for the next chunk to attend to
        dict(name="append-8x2k", kind="append", seqs=8, lo=501, hi=4000, q=4000, hq=8, heads=8, d=128, page=64, rounds=1, type="bfloat16"),
        # a step of a beam search: the old beams go, four of each prompt are forked, and take a token each
        dict(name="pages-beams", kind="pages", act="beams", seqs=16, lo=100, hi=4000, ways=4, layers=2, heads=8, d=128, page=64),
        # sequences copied, the old ones freed, and the pool made dense again
        dict(name="pages-compact", kind="pages", act="compact", seqs=8, lo=4000, hi=12000, ways=1, layers=2, heads=8, d=128, page=64),
        # one short prompt: latency
        dict(name="prompt-333", kind="prompt", seqs=1, lo=333, hi=333, prefix=0, hq=8, heads=2, d=64, causal=True, type="float16"),
        # prompts as they arrive, packed; every other one continues a prefix that was read back
        dict(name="prompt-packed", kind="prompt", seqs=7, lo=120, hi=2047, prefix=1000, hq=32, heads=8, d=128, causal=True, type="bfloat16"),
        # one long prompt
        dict(name="prompt-8192", kind="prompt", seqs=1, lo=8192, hi=8192, prefix=0, hq=32, heads=8, d=128, causal=True, type="bfloat16"),
        # texts to be embedded: an encoder sees them whole
        dict(name="prompt-encoder", kind="prompt", seqs=48, lo=16, hi=512, prefix=0, hq=12, heads=12, d=64, causal=False, type="float16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "append", "pages", "prompt", "prompt"])
    d = rng.choice([64, 128, 128, 256])
    page = rng.choice([32, 64, 64, 128])
    heads = rng.choice([1, 2, 4, 8, 8, 12])
    typ = rng.choice(["float16", "bfloat16"])
    if kind == "attend":
        group = rng.choice([1, 2, 3, 4, 5, 8, 16])
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, max(2, min(100_000, 300_000_000 // (seqs * heads * d * (2 if group < 8 else 4)))))
        return dict(kind=kind, seqs=seqs, lo=max(1, int(hi * rng.random())), hi=hi, q=rng.choice([1, 1, 1, 2, 4, 9]),
                    hq=heads * group, heads=heads, d=d, page=page, rounds=rng.choice([1, 1, 3]), type=typ)
    if kind == "append":
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, max(2, 16_000_000 // (seqs * heads * d)))
        return dict(kind=kind, seqs=seqs, lo=max(1, int(hi * rng.random())), hi=hi, q=rng.choice([1, 3, hi, hi]), hq=heads, heads=heads,
                    d=d, page=page, rounds=rng.choice([1, 1, 2, 3]), type=typ)
    if kind == "pages":
        act = rng.choice(["beams", "compact"])
        seqs = _log(rng, 1, 24)
        hi = _log(rng, 2, max(3, 48_000_000 // (seqs * heads * d)))
        return dict(kind=kind, act=act, seqs=seqs, lo=max(1, int(hi * rng.random())), hi=hi, ways=rng.choice([1, 2, 4]) if act == "beams" else 1,
                    layers=rng.choice([1, 2, 3]), heads=heads, d=d, page=page)
    d = rng.choice([64, 128, 128])
    group = rng.choice([1, 2, 3, 4, 8])
    seqs = _log(rng, 1, 48)
    hi = _log(rng, 1, max(2, int(min(8192, math.sqrt(5e10 / (seqs * heads * group * d))))))
    return dict(kind=kind, seqs=seqs, lo=max(1, int(hi * rng.random())), hi=hi, prefix=rng.choice([0, 0, _log(rng, 1, hi)]), hq=heads * group,
                heads=heads, d=d, causal=rng.random() < 0.7, type=typ)


def _lengths(case):
    """The sequences' lengths: spread evenly in their logarithm, in no order."""
    n, lo, hi = case["seqs"], case["lo"], case["hi"]
    got = [hi if n == 1 else int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]
    random.Random(n).shuffle(got)
    return got


def _rows(case):
    """How many of each sequence's tokens are this call's."""
    return [min(x, 1 + (i * 7 + case["q"] - 1) % case["q"]) if case["kind"] == "attend" else min(x, case["q"]) for i, x in enumerate(_lengths(case))]


def _prefixes(case):
    return [case["prefix"] if i % 2 else 0 for i in range(case["seqs"])]


def work(case):
    lens, d, heads = _lengths(case), case["d"], case["heads"]
    row = d + 8  # a token of a head in the cache: keys and values
    if case["kind"] == "attend":
        rows = _rows(case)
        pairs = sum(n * x - n * (n - 1) // 2 for n, x in zip(rows, lens))
        return {"bytes": sum(lens) * heads * row + 4 * sum(rows) * case["hq"] * d, "flops": 4 * pairs * case["hq"] * d}
    if case["kind"] == "append":
        n = sum(_rows(case)) * heads
        return {"bytes": 2 * n * (row + 4 * d), "flops": 4 * n * (case["rounds"] * d * math.log2(d) + 6 * d)}
    if case["kind"] == "pages":
        size = case["layers"] * heads * case["page"] * row
        if case["act"] == "beams":
            n = sum(1 for x in lens if x % case["page"]) * case["ways"]
            return {"bytes": 2 * n * size + 12 * case["ways"] * sum(-(-x // case["page"]) for x in lens), "flops": 0}
        return {"bytes": 4 * size * sum(-(-x // case["page"]) for x in lens), "flops": 0}
    pre = _prefixes(case)
    pairs = sum(n * (n + p) - (n * (n - 1) // 2 if case["causal"] else 0) for n, p in zip(lens, pre))
    return {"bytes": 2 * d * (2 * sum(lens) * case["hq"] + 2 * (sum(lens) + sum(pre)) * heads), "flops": 4 * pairs * case["hq"] * d}


# ------------------------------------------------------------------ inputs

def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(counts):
    return _int([sum(counts[:i]) for i in range(len(counts) + 1)])


def _signs(case, g):
    return torch.randint(0, 2, (case.get("rounds", 1), case["d"]), generator=g, device=DEV).float() * 2 - 1


def _pool(case, g, layers, pages):
    """Pages full of tokens, quantised as a Gaussian row is."""
    d, heads, tiles = case["d"], case["heads"], case["page"] // TILE
    pool = torch.empty(layers, pages, heads, tiles, TILE * (d + 8), dtype=torch.uint8, device=DEV)
    codes = lambda: (torch.randn(pages, heads, tiles, TILE * d, generator=g, device=DEV) / STEP).floor_().add_(8).clamp_(0, 15).to(torch.uint8)  # noqa: E731
    scales = lambda s: (s * STEP * torch.exp(0.3 * torch.randn(pages, heads, tiles, TILE, generator=g, device=DEV))).view(torch.uint8)  # noqa: E731
    for layer in range(layers):
        for at, size in ((0, 1.5), (TILE * (d // 2 + 4), 1.0)):
            c = codes()
            pool[layer, ..., at:at + TILE * d // 2] = c[..., 0::2] | (c[..., 1::2] << 4)
            pool[layer, ..., at + TILE * d // 2:at + TILE * (d // 2 + 4)] = scales(size)
    return pool


def _cache(case, g, lens, slots, spare=0, layers=1, signs=None, spread=True):
    """A pool and its tables, the sequences' pages wherever a server's history left them."""
    have = [-(-x // case["page"]) for x in lens]
    used, width = sum(have), max(have) + 1
    pages = used + spare + (used // 8 if spread else 0)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32) if spread else torch.arange(pages, dtype=torch.int32, device=DEV)
    table = torch.full((slots, width), -1, dtype=torch.int32, device=DEV)
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(have):
        table[i, :n] = order[at:at + n]
        at += n
    refs[order[:used].long()] = 1
    full = torch.zeros(slots, dtype=torch.int32, device=DEV)
    full[:len(lens)] = _int(list(lens))
    signs = _signs(case, g) if signs is None else signs
    s = dict(pool=_pool(case, g, layers, pages), table=table, lens=full, refs=refs, signs=signs, page=case["page"])
    if own:
        from ultravec_ann_b200_loader import load

        s["cache"] = load().KvCache.over(s["pool"], table, full, refs, signs=signs, head_dim=case["d"], page_tokens=case["page"])
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, lens, d = case["kind"], _lengths(case), case["d"]
    if kind in ("attend", "append"):
        rows = _rows(case)
        s = _cache(case, g, lens, case["seqs"] + 1)
        s |= dict(seqs=_int(list(range(case["seqs"]))[::-1]), rows=_starts(rows[::-1]), most=max(rows), total=sum(rows))
        typ = getattr(torch, case["type"])
        if kind == "attend":
            s["q"] = torch.randn(sum(rows), case["hq"], d, generator=g, device=DEV).to(typ)
        else:  # keys have channels that stand out, and a mean; values have neither
            loud = torch.exp(0.7 * torch.randn(case["heads"], d, generator=g, device=DEV))
            mean = loud * torch.randn(case["heads"], d, generator=g, device=DEV)
            s["k"] = (torch.randn(sum(rows), case["heads"], d, generator=g, device=DEV) * loud + mean).to(typ)
            s["v"] = torch.randn(sum(rows), case["heads"], d, generator=g, device=DEV).to(typ)
    elif kind == "pages":
        n, ways = case["seqs"], case["ways"]
        spare = sum(-(-x // case["page"]) for x in lens) if case["act"] == "compact" else n * ways
        s = _cache(case, g, lens, n * (1 + ways), spare, case["layers"], spread=case["act"] == "beams")
        s |= dict(src=_int([i for i in range(n) for _ in range(ways)]), dst=_int(list(range(n, n * (1 + ways)))), one=_int([1] * (n * ways)))
    else:
        pre = _prefixes(case)
        keys = [n + p for n, p in zip(lens, pre)]
        typ = getattr(torch, case["type"])
        make = lambda n, h: torch.randn(n, h, d, generator=g, device=DEV)  # noqa: E731
        s = dict(q=(1.5 * make(sum(lens), case["hq"])).to(typ), k=make(sum(keys), case["heads"]).to(typ), v=make(sum(keys), case["heads"]).to(typ),
                 starts_q=_starts(lens), starts_k=_starts(keys), longest_q=max(lens), longest_k=max(keys))
    return dict(s, kind=kind, act=case.get("act"), causal=case.get("causal"))


# ------------------------------------------------------------------ one pass

def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "attend":
        return _attend(s)
    if s["kind"] == "append":
        return _append(s)
    if s["kind"] == "pages":
        return _beams(s) if s["act"] == "beams" else _defragment(s)
    return _prompt(s)


def _run_own(s):
    if s["kind"] == "attend":
        return s["cache"].attend(s["seqs"], s["q"], starts=s["rows"], most=s["most"])
    if s["kind"] == "append":
        s["cache"].append(s["seqs"], s["k"], s["v"], starts=s["rows"])
        return s["cache"].read(s["seqs"], s["rows"], s["total"], dtype=s["k"].dtype)
    if s["kind"] == "pages":
        c = s["cache"]
        if s["act"] == "beams":
            c.free(s["dst"])
            c.fork(s["src"], s["dst"])
            c.extend(s["dst"], s["one"])
        else:
            c.copy(s["src"], s["dst"])
            c.free(s["src"])
            c.compact()
            c.fork(s["dst"], s["src"])
            c.free(s["dst"])
        return s["table"], s["lens"], s["refs"], s["pool"]
    from ultravec_ann_b200_loader import load

    return load().prompt_attention(s["q"], s["k"], s["v"], s["starts_q"], s["starts_k"], causal=s["causal"])


def _rotation(signs):
    """R with y = x R^T, as a matrix."""
    d = signs.shape[1]
    i = torch.arange(d, device=signs.device)
    odd = i[:, None] & i[None, :]
    odd = odd ^ (odd >> 4)
    odd = odd ^ (odd >> 2)
    odd = (odd ^ (odd >> 1)) & 1
    h = (1 - 2 * odd).float() / math.sqrt(d)
    r = h * signs[0]
    for more in signs[1:]:
        r = (h * more) @ r
    return r


def _values(codes):
    """Rows of packed codes as n - 7.5."""
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 7.5


def _unpack(tiles, d):
    """Keys and values, rotated, of tiles [..., 32 (d + 8)] as [..., 32, d]."""
    lead, half = tiles.shape[:-1], TILE * (d // 2)
    k = _values(tiles[..., :half].reshape(*lead, TILE, d // 2)) * tiles[..., half:half + 4 * TILE].contiguous().view(torch.float32)[..., None]
    at = half + 4 * TILE
    v = tiles[..., at:at + half].reshape(*lead, TILE // 2, d // 4, 2, 2).transpose(-2, -3).reshape(*lead, TILE, d // 2)
    return k, _values(v) * tiles[..., at + half:].contiguous().view(torch.float32)[..., None]


def _held(s, d):
    """Keys and values of every listed sequence, rotated: [sequences, heads, tokens, d]."""
    pages = s["table"][s["seqs"].long()].clamp(min=0).long()
    tiles = s["pool"][0][pages].transpose(1, 2)  # sequences, heads, pages, tiles, bytes
    k, v = _unpack(tiles, d)
    return k.flatten(2, 4), v.flatten(2, 4)


def _places(starts, most):
    """For packed rows: which of [sequences, most] are rows, and which row each is."""
    n = (starts[1:] - starts[:-1]).long()
    i = torch.arange(most, device=starts.device)
    return i[None, :] < n[:, None], (starts[:-1].long()[:, None] + i).clamp(max=max(int(starts[-1]) - 1, 0))


def _attend(s):
    q, d = s["q"], s["q"].shape[2]
    k, v = _held(s, d)
    group = q.shape[1] // k.shape[1]
    r = _rotation(s["signs"])
    live, at = _places(s["rows"], s["most"])
    x = (q.float() @ r.T)[at].unflatten(2, (-1, group))  # sequences, rows, heads, group, d
    x = x.permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = x @ k.transpose(2, 3) / math.sqrt(d)
    lens, n = s["lens"][s["seqs"].long()].long(), live.sum(1)
    last = (lens - n)[:, None] + torch.arange(s["most"], device=q.device)
    seen = torch.arange(k.shape[2], device=q.device)[None, None, :] <= last[:, :, None]
    seen = seen[:, None, None].expand(-1, k.shape[1], group, -1, -1).flatten(2, 3)
    p = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
    v = v.masked_fill((torch.arange(k.shape[2], device=q.device) >= lens[:, None])[:, None, :, None], 0)
    out = ((p @ v) @ r).unflatten(2, (group, -1)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[live].to(q.dtype)


def _quantise(x, r):
    """Codes n - 7.5 and scales of rows."""
    x = x.float()
    e = torch.frexp(x.abs().amax(-1, keepdim=True)).exponent
    y = torch.ldexp(x, -e) @ r.T
    square = (y * y).sum(-1, keepdim=True)
    some = square > 0  # a row of zeros has the scale zero
    level = torch.where(some, torch.floor(y / (STEP * torch.sqrt(square / y.shape[-1]))), 0).clamp(-8, 7) + 0.5
    return level, torch.ldexp(torch.where(some, square / (level * y).sum(-1, keepdim=True), 0), e)


def _append(s):
    d, page = s["k"].shape[2], s["page"]
    r = _rotation(s["signs"])
    live, at = _places(s["rows"], s["most"])
    seqs = s["seqs"].long()
    n = live.sum(1)
    token = ((s["lens"][seqs].long() - n)[:, None] + torch.arange(s["most"], device=live.device))[live]
    where = s["table"][seqs.repeat_interleave(n), token // page].long()
    tile, row = token % page // TILE, token % TILE
    half = TILE * (d // 2)
    wide = torch.arange(d // 2, device=live.device)
    for x, base in ((s["k"], 0), (s["v"], half + 4 * TILE)):
        level, scale = _quantise(x, r)
        code = (level + 7.5).to(torch.uint8)
        code = code[..., 0::2] | (code[..., 1::2] << 4)
        byte = base + (row[:, None] * (d // 2) + wide if base == 0 else (row // 2)[:, None] * d + wide // 2 * 4 + (row % 2)[:, None] * 2 + wide % 2)
        pool = s["pool"][0]
        heads = torch.arange(code.shape[1], device=live.device)
        pool[where[:, None, None], heads[None, :, None], tile[:, None, None], byte[:, None, :]] = code
        byte = base + half + 4 * row[:, None] + torch.arange(4, device=live.device)
        pool[where[:, None, None], heads[None, :, None], tile[:, None, None], byte[:, None, :]] = scale.contiguous().view(torch.uint8)
    tiles = s["pool"][0][where, :, tile]  # rows, heads, bytes
    k, v = _unpack(tiles, d)
    line = torch.arange(len(row), device=live.device)
    k, v = k[line, :, row], v[line, :, row]
    return (k @ r).to(s["k"].dtype), (v @ r).to(s["k"].dtype)


def _count(tokens, page):
    return (tokens + page - 1) // page


def _free(s, seqs):
    seqs = seqs.long()
    rows = s["table"][seqs]
    gone = rows[rows >= 0].long()
    s["refs"].index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    s["table"][seqs] = -1
    s["lens"][seqs] = 0


def _fork(s, src, dst):
    src, dst = src.long(), dst.long()
    rows = s["table"][src]
    s["table"][dst] = rows
    s["lens"][dst] = s["lens"][src]
    more = rows[rows >= 0].long()
    s["refs"].index_add_(0, more, torch.ones_like(more, dtype=torch.int32))


def _take(s, seqs, first, n):
    """n[i] fresh pages, the lowest free ones in the order of the list, into the table from column first[i] on."""
    total = int(n.sum())
    fresh = (s["refs"] == 0).nonzero()[:total, 0]
    who = torch.repeat_interleave(torch.arange(len(n), device=n.device), n)
    at = torch.arange(total, device=n.device) - (n.cumsum(0) - n)[who]
    s["table"][seqs[who], first[who] + at] = fresh.to(torch.int32)
    s["refs"][fresh] = 1
    return fresh, who, at


def _extend(s, seqs, counts):
    seqs, counts, page = seqs.long(), counts.long(), s["page"]
    lens = s["lens"][seqs].long()
    have = _count(lens, page)
    last = s["table"][seqs, (have - 1).clamp(min=0)].long()
    shared = (counts > 0) & (lens % page != 0) & (s["refs"][last.clamp(min=0)] > 1)
    fresh, who, at = _take(s, seqs, have - shared.long(), _count(lens + counts, page) - have + shared.long())
    new = fresh[shared[who] & (at == 0)]
    old = last[shared]
    s["pool"][:, new] = s["pool"][:, old]
    s["refs"].index_add_(0, old, torch.full_like(old, -1, dtype=torch.int32))
    s["lens"][seqs] = (lens + counts).to(torch.int32)


def _beams(s):
    _free(s, s["dst"])
    _fork(s, s["src"], s["dst"])
    _extend(s, s["dst"], s["one"])
    return s["table"], s["lens"], s["refs"], s["pool"]


def _defragment(s):
    src, dst = s["src"].long(), s["dst"].long()
    have = _count(s["lens"][src].long(), s["page"])
    fresh, who, at = _take(s, dst, torch.zeros_like(have), have)
    s["pool"][:, fresh] = s["pool"][:, s["table"][src[who], at].long()]
    s["lens"][dst] = s["lens"][src]
    _free(s, s["src"])
    used = s["refs"] > 0
    n = int(used.sum())
    high, low = used[n:].nonzero()[:, 0] + n, (~used[:n]).nonzero()[:, 0]
    to = torch.arange(len(used), dtype=torch.int32, device=used.device)
    to[high] = low.to(torch.int32)
    s["pool"][:, low] = s["pool"][:, high]
    s["refs"][low] = s["refs"][high]
    s["refs"][high] = 0
    s["table"].copy_(torch.where(s["table"] >= 0, to[s["table"].clamp(min=0).long()], s["table"]))
    _fork(s, s["dst"], s["src"])
    _free(s, s["dst"])
    return s["table"], s["lens"], s["refs"], s["pool"]


def _prompt(s):
    q, d = s["q"], s["q"].shape[2]
    live, at = _places(s["starts_q"], s["longest_q"])
    some, from_ = _places(s["starts_k"], s["longest_k"])
    group = q.shape[1] // s["k"].shape[1]
    x = q.float()[at].unflatten(2, (-1, group)).permute(0, 2, 3, 1, 4)  # sequences, heads, group, rows, d
    k, v = (t.float()[from_].permute(0, 2, 1, 3)[:, :, None] for t in (s["k"], s["v"]))
    v = v.masked_fill(~some[:, None, None, :, None], 0)
    score = x @ k.transpose(3, 4)
    score *= 1 / math.sqrt(d)
    seen = some[:, None, :]
    if s["causal"]:
        i = torch.arange(s["longest_q"], device=q.device)[None, :] + (some.sum(1) - live.sum(1))[:, None]
        seen = seen & (torch.arange(s["longest_k"], device=q.device) <= i[:, :, None])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    out = torch.softmax(score, -1) @ v
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)[live].to(q.dtype)


# ------------------------------------------------------------------ from the definitions, in 64 bits

def _back(y, signs):
    """R^T y, in the stages of the transform."""
    d = y.shape[-1]
    for sign in signs.flip(0):
        h = 1
        while h < d:
            y = y.reshape(*y.shape[:-1], d // (2 * h), 2, h) if y.shape[-1] == d else y
            y = torch.stack((y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]), -2)
            y = y.reshape(*y.shape[:-3], d)
            h *= 2
        y = y * sign / math.sqrt(d)
    return y


def _forth(x, signs):
    d = x.shape[-1]
    for sign in signs:
        x = _back((x * sign), torch.ones(1, d, dtype=x.dtype, device=x.device))
    return x


def exact(case, seed):
    if case["kind"] == "pages":
        return None
    s = prepare(case, seed)
    d = case["d"]
    signs = s["signs"].double() if "signs" in s else None
    if case["kind"] == "append":
        got = []
        for x in (s["k"], s["v"]):
            y = _forth(x.double(), signs)
            square = (y * y).sum(-1, keepdim=True)
            level = (torch.floor(y / (STEP * (square / d).sqrt())).clamp(-8, 7)) + 0.5
            got.append(_back(level * square / (level * y).sum(-1, keepdim=True), signs))
        return tuple(got)
    if case["kind"] == "prompt":
        q, k, v, outs = s["q"].double(), s["k"].double(), s["v"].double(), torch.empty_like(s["q"], dtype=torch.float64)
        a, b = s["starts_q"].tolist(), s["starts_k"].tolist()
        for i in range(len(a) - 1):
            n, m = a[i + 1] - a[i], b[i + 1] - b[i]
            hide = torch.ones(n, m, dtype=torch.bool, device=q.device).triu(m - n + 1) if case["causal"] else None
            for h in range(case["hq"]):
                j = h // (case["hq"] // case["heads"])
                e = q[a[i]:a[i + 1], h] @ k[b[i]:b[i + 1], j].T / math.sqrt(d)
                e = e if hide is None else e.masked_fill(hide, -math.inf)
                e = (e - e.amax(1, keepdim=True)).exp()
                outs[a[i]:a[i + 1], h] = e @ v[b[i]:b[i + 1], j] / e.sum(1, keepdim=True)
        return outs
    x, outs, starts = _forth(s["q"].double(), signs), [], s["rows"].tolist()
    half = TILE * (d // 2)
    for i, seq in enumerate(s["seqs"].tolist()):
        n, rows = int(s["lens"][seq]), x[starts[i]:starts[i + 1]]
        tiles = s["pool"][0, s["table"][seq, :-(-n // case["page"])].long()].transpose(0, 1).flatten(1, 2)  # heads, tiles, bytes
        held = []
        for at in (0, half + 4 * TILE):
            c = tiles[..., at:at + half]
            if at:
                c = c.reshape(*c.shape[:2], TILE // 2, d // 4, 2, 2).permute(0, 1, 2, 4, 3, 5)
            c = c.reshape(case["heads"], -1, d // 2)
            scale = tiles[..., at + half:at + half + 4 * TILE].contiguous().view(torch.float32).reshape(case["heads"], -1, 1).double()
            y = torch.empty(case["heads"], c.shape[1], d, dtype=torch.float64, device=c.device)
            y[..., 0::2], y[..., 1::2] = (c & 15) - 7.5, (c >> 4) - 7.5
            held.append((y * scale)[:, :n])
        k, v = held
        r = rows.unflatten(1, (case["heads"], -1)).permute(1, 2, 0, 3)  # heads, group, rows, d
        e = r @ k.transpose(1, 2)[:, None] / math.sqrt(d)
        m = rows.shape[0]
        e = e.masked_fill(torch.ones(m, n, dtype=torch.bool, device=e.device).triu(n - m + 1), -math.inf)
        e = (e - e.amax(-1, keepdim=True)).exp()
        o = (e @ v[:, None]) / e.sum(-1, keepdim=True)
        outs.append(_back(o, signs).permute(2, 0, 1, 3).flatten(1, 2))
    return torch.cat(outs)
