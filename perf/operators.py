"""Cases of the 4-bit KV cache and of the token log-probabilities.

A serving step of many requests over a paged cache whose keys and values are
held in 4 bits:

  reserve    block tables, slot maps and positions of the new tokens from the
             requests' lengths (nimf.KV4Cache.reserve)
  append     rotary embedding of the new queries and keys, keys and values
             quantised into their slots (nimf.KV4Cache.append), the rows read
             back as the values that they stand for (nimf.KV4Cache.read)
  attention  causal attention of the new tokens over the cache
             (nimf.KV4Cache.attention)
  logprobs   log-probabilities of given tokens, the entropy of each row and
             its most likely alternatives (nimf.logprobs_dev)

run() computes them from elementary torch operations where `own` is false, and
by the library's calls where it is true.

The cache is uint8 [blocks][kv heads][block / 16][tile], a tile being 16 tokens
of one head:

  K codes [16][dim / 2], V codes [16][dim / 2],
  K {scale, minimum} float32 [dim / group][16][2], V {scale, minimum} the same

A group of `group` channels of one token and head is coded as
scale = (max - min) / 15, code = min(15, round((x - min) / scale)), and stands
for code * scale + min; every step is rounded to float32.  Channel d of a key
is nibble d % 8 (the low one of a byte first) of the 32-bit word
(d % 32 / 8) * (dim / 32) + d / 32 of its row; of a value, nibble
d % 4 + 4 * (d % 64 / 32) of word (d % 32 / 4) * (dim / 64) + d / 64.
"""
import math
import random
import sys

import torch

own = False

TILE = 16


# ----------------------------------------------------------------- the cases
def listed():
    return [
        # one new token for each of 64 running requests: a decode step's bookkeeping
        dict(name="reserve step", op="reserve", seqs=64, low=1, high=4095, new_low=1, new_high=1, block=16, width=256, spare=8),
        # 256 prompts of ragged lengths admitted at once, the pool running dry before the last ones
        dict(name="reserve prompts", op="reserve", seqs=256, low=0, high=700, new_low=1, new_high=1500, block=32, width=80, spare=-900),
        # one new token each of 64 requests, the 7B attention's 32 heads of 128
        dict(name="append step", op="append", rows=64, pad=0, heads=32, kv_heads=32, dim=128, group=128, block=16, max_seq=4096),
        # prompts of 8,000 tokens in all, grouped heads, fine groups, the batch padded by 100 rows
        dict(name="append prompts", op="append", rows=8100, pad=100, heads=32, kv_heads=8, dim=128, group=32, block=32, max_seq=9000),
        # one request decoding, 7B heads: latency
        dict(name="decode one", op="attention", seqs=1, low=519, high=519, prompt=1, heads=32, kv_heads=32, dim=128, group=128, block=16),
        # 64 requests of ragged lengths, grouped heads
        dict(name="decode batch", op="attention", seqs=64, low=1, high=4096, prompt=1, heads=32, kv_heads=8, dim=128, group=64, block=16),
        # a few requests with long contexts
        dict(name="decode long", op="attention", seqs=4, low=65537, high=131000, prompt=1, heads=32, kv_heads=8, dim=128, group=128, block=64),
        # a chunk of 2,048 prompt tokens after 4,096 cached ones, 7B heads
        dict(name="prompt chunk", op="attention", seqs=1, low=6144, high=6144, prompt=2048, heads=32, kv_heads=32, dim=128, group=128, block=32),
        # 32 requests decoding while another's prompt of 777 tokens runs along
        dict(name="mixed step", op="attention", seqs=33, low=777, high=2000, prompt=777, heads=16, kv_heads=4, dim=64, group=32, block=16),
        # the token just chosen by one request, vocabulary of the 7B model
        dict(name="logprobs one", op="logprobs", rows=1, vocab=32000, top=5, masked=0),
        # a decode batch, a large odd vocabulary, every fourth row limited to a few tokens
        dict(name="logprobs batch", op="logprobs", rows=64, vocab=128001, top=20, masked=1),
        # scoring a prompt of 4,096 tokens
        dict(name="logprobs prompt", op="logprobs", rows=4096, vocab=32000, top=1, masked=0),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["reserve", "append", "attention", "attention", "attention", "logprobs"])
    if op == "reserve":
        block = rng.choice([16, 32, 64, 128])
        high, new = _log_int(rng, 1, 4000), _log_int(rng, 1, 1500)
        seqs = _log_int(rng, 1, 1000) if new < 64 else _log_int(rng, 1, 250)
        return dict(op=op, seqs=seqs, low=0, high=high, new_low=rng.choice([0, 1]), new_high=new, block=block,
                    width=-(-(high + new) // block) + rng.choice([0, 0, 1, 7]), spare=rng.choice([-20, -1, 0, 3, 100]))
    if op == "append":
        dim = rng.choice([64, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 8, 32])
        heads = kv * rng.choice([1, 2, 4, 7] if kv < 32 else [1])
        rows = _log_int(rng, 1, max(2, min(9000, 8100 * (32 + 16) * 128 // ((heads + 2 * kv) * dim))))
        return dict(op=op, rows=rows, pad=rng.choice([0, 1, 37]) % rows, heads=heads, kv_heads=kv, dim=dim,
                    group=rng.choice([g for g in (32, 64, 128) if dim % g == 0]), block=rng.choice([16, 32, 64]), max_seq=9000 + rng.randrange(900))
    if op == "attention":
        dim = rng.choice([64, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 8, 32])
        heads = kv * (rng.choice([1, 2, 4, 7, 8]) if kv < 32 else 1)
        case = dict(op=op, seqs=1, low=1, high=1, prompt=1, heads=heads, kv_heads=kv, dim=dim,
                    group=rng.choice([g for g in (32, 64, 128) if dim % g == 0]), block=rng.choice([16, 32, 64, 128]))
        if rng.random() < 0.65:  # a decode step: up to 400,000 tokens of 8 heads of 128 are in the cache
            case["high"] = _log_int(rng, 1, 100000)
            case["low"] = rng.choice([1, max(1, case["high"] // 2), case["high"]])
            most = 400000 * 1024 // (kv * dim * case["high"])
            case["seqs"] = _log_int(rng, 1, max(1, min(300, most)))
        else:  # a prompt or a chunk of one, alone or beside decoding requests
            case["prompt"] = _log_int(rng, 2, 2000)
            case["high"] = case["prompt"] + rng.choice([0, _log_int(rng, 1, 4000)])
            most = 32 * 2048 * 6144 // (heads * case["prompt"] * case["high"])
            case["seqs"] = max(1, min(24, _log_int(rng, 1, max(1, most))))
            case["low"] = max(1, case["high"] // 3)
        return case
    vocab = _log_int(rng, 40, 260000)
    rows = _log_int(rng, 1, max(1, min(5000, 4096 * 32000 // vocab)))
    return dict(op=op, rows=rows, vocab=vocab, top=rng.choice([0, 1, 5, 20, 32]), masked=rng.choice([0, 0, 1]))


# ------------------------------------------------------- lengths of the cases
def _lengths(case):
    """Cached tokens and new tokens of each request of an attention case: the
    first has the case's longest context (and its prompt), the others ragged
    ones."""
    rng = random.Random("%s" % sorted((k, v) for k, v in case.items() if k not in ("name",)))
    lens = [case["high"]] + [_log_int(rng, case["low"], case["high"]) for _ in range(case["seqs"] - 1)]
    new = [case["prompt"]] + [1] * (case["seqs"] - 1)
    return lens, new


def _requests(case):
    """Cached tokens, new tokens and free blocks of a reserve case."""
    rng = random.Random("%s" % sorted((k, v) for k, v in case.items() if k not in ("name",)))
    n, bs = case["seqs"], case["block"]
    lens = [rng.randint(case["low"], case["high"]) for _ in range(n)]
    new = [rng.randint(case["new_low"], case["new_high"]) for _ in range(n)]
    need = sum(-(-(a + b) // bs) - -(-a // bs) for a, b in zip(lens, new))
    have = sum(-(-a // bs) for a in lens)
    return lens, new, have, max(0, need + case["spare"])


def _tile_bytes(case):
    return TILE * case["dim"] + 2 * TILE * 8 * (case["dim"] // case["group"])


def work(case):
    op = case["op"]
    if op == "reserve":
        lens, new, have, free = _requests(case)
        rows = sum(new)
        taken = min(free, sum(-(-(a + b) // case["block"]) - -(-a // case["block"]) for a, b in zip(lens, new)))
        return {"bytes": 4 * (5 * len(lens) + 2 * taken + 2 * rows), "flops": 0}
    if op == "append":
        t, d = case["rows"], case["dim"]
        read = 4 * t * d * (case["heads"] + 2 * case["kv_heads"]) + 8 * t + 8 * t * (d // 2)
        written = 4 * t * d * (case["heads"] + 2 * case["kv_heads"]) + t * case["kv_heads"] * _tile_bytes(case) // TILE
        return {"bytes": read + written, "flops": 3 * t * d * (case["heads"] + case["kv_heads"]) + 10 * t * d * case["kv_heads"]}
    if op == "attention":
        lens, new = _lengths(case)
        cached = sum(lens) * case["kv_heads"] * _tile_bytes(case) // TILE
        seen = sum(n * (a - n) + n * (n + 1) // 2 for a, n in zip(lens, new))
        return {"bytes": cached + 8 * sum(new) * case["heads"] * case["dim"] + 4 * sum(-(-a // case["block"]) for a in lens),
                "flops": 4 * seen * case["heads"] * case["dim"]}
    r, v = case["rows"], case["vocab"]
    return {"bytes": 4 * r * v + 16 * r + 8 * r * case["top"], "flops": 4 * r * v}


# ------------------------------------------------ the cache format, plain torch
def _code(x, group):
    """x [..., dim] float32 as codes [..., dim] uint8, scale and minimum
    [..., dim / group]."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // group, group)
    low, high = g.amin(-1), g.amax(-1)
    scale = (high - low) / torch.full_like(low, 15.0)
    code = torch.round((g - low[..., None]) / torch.where(scale > 0, scale, 1.0)[..., None]).clamp_(0, 15)
    return code.to(torch.uint8).reshape(x.shape), scale, low


def _value(code, scale, low):
    g = code.reshape(*scale.shape, -1).float()
    return (g * scale[..., None] + low[..., None]).reshape(code.shape)


def _pack(code, key):
    """Codes [..., dim] in the order in which a row holds them, two a byte."""
    d, lead = code.shape[-1], code.shape[:-1]
    if key:
        c = code.reshape(*lead, d // 32, 4, 8).transpose(-3, -2)
    else:
        c = code.reshape(*lead, d // 64, 2, 8, 4).movedim(-2, len(lead))
    c = c.reshape(*lead, d // 2, 2)
    return c[..., 0] | (c[..., 1] << 4)


def _unpack(rows, key):
    """_pack's inverse: bytes [..., dim / 2] as codes [..., dim]."""
    d, lead = rows.shape[-1] * 2, rows.shape[:-1]
    c = torch.stack((rows & 15, rows >> 4), -1)
    if key:
        c = c.reshape(*lead, 4, d // 32, 8).transpose(-3, -2)
    else:
        c = c.reshape(*lead, 8, d // 64, 2, 4).movedim(len(lead), -2)
    return c.reshape(*lead, d)


def _open(tiles, dim, group):
    """Tiles [..., tile bytes] as the keys and values [..., 16, dim] float32
    that they stand for."""
    lead, half, par = tiles.shape[:-1], TILE * dim // 2, TILE * 8 * (dim // group)
    got = []
    for key, codes, at in ((True, 0, 2 * half), (False, half, 2 * half + par)):
        c = _unpack(tiles[..., codes:codes + half].reshape(*lead, TILE, dim // 2), key)
        p = tiles[..., at:at + par].contiguous().view(torch.float32).reshape(*lead, dim // group, TILE, 2).transpose(-3, -2)
        got.append(_value(c, p[..., 0], p[..., 1]))
    return got


def _random_cache(gen, blocks, case):
    """A pool whose every block holds keys and values as they come out of a
    projection: normal, some channels of the keys much larger than the others."""
    kv, dim, group = case["kv_heads"], case["dim"], case["group"]
    tiles = case["block"] // TILE
    half, par = TILE * dim // 2, TILE * 8 * (dim // group)
    cache = torch.empty(blocks, kv, tiles, _tile_bytes(case), dtype=torch.uint8, device="cuda")
    wide = 1 + 4 * (torch.rand(kv, 1, 1, dim, generator=gen, device="cuda") < 0.03)
    step = max(1, (1 << 26) // (kv * case["block"] * dim))
    for at in range(0, blocks, step):
        part = cache[at:at + step]
        for key, codes, params in ((True, 0, 2 * half), (False, half, 2 * half + par)):
            x = torch.randn(part.shape[0], kv, tiles, TILE, dim, generator=gen, device="cuda")
            code, scale, low = _code(x * wide if key else x, group)
            part[..., codes:codes + half] = _pack(code, key).flatten(-2)
            both = torch.stack((scale, low), -1).transpose(-3, -2).contiguous()
            part[..., params:params + par] = both.flatten(-3).view(torch.uint8)
    return cache


# -------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    s = dict(case=case)
    op = case["op"]
    if op == "reserve":
        lens, new, have, free = _requests(case)
        bs, n = case["block"], case["seqs"]
        blocks = have + free
        order = torch.randperm(max(1, blocks), generator=gen, device="cuda").int()
        pages = torch.tensor([-(-a // bs) for a in lens], device="cuda")
        start = torch.cumsum(pages, 0) - pages
        col = torch.arange(case["width"], device="cuda")
        at = (start[:, None] + col).clamp(max=max(0, blocks - 1))
        s.update(table=torch.where(col < pages[:, None], order[at], -1).int(), lens=ints(lens), new=ints(new),
                 free=torch.cat((order[have:], order[:have])).contiguous(), n_free=ints([free]), blocks=max(1, blocks),
                 rows=sum(new) + 5)
    elif op == "append":
        t, d, kv = case["rows"], case["dim"], case["kv_heads"]
        blocks = -(-t // case["block"]) + 3
        s.update(q=torch.randn(t, case["heads"], d, generator=gen, device="cuda"),
                 k=torch.randn(t, kv, d, generator=gen, device="cuda") * (1 + 4 * (torch.rand(kv, d, generator=gen, device="cuda") < 0.03)),
                 v=torch.randn(t, kv, d, generator=gen, device="cuda"), blocks=blocks,
                 slots=torch.randperm(blocks * case["block"], generator=gen, device="cuda")[:t].int(),
                 positions=torch.randint(0, case["max_seq"], (t,), generator=gen, device="cuda").int(),
                 cache=torch.zeros(blocks, kv, case["block"] // TILE, _tile_bytes(case), dtype=torch.uint8, device="cuda"))
        if case["pad"]:
            s["slots"][-case["pad"]:] = -1
        inv = 1.0 / 10000.0 ** (torch.arange(d // 2, device="cuda").float() / (d // 2))
        ang = torch.arange(case["max_seq"], device="cuda").float()[:, None] * inv
        s.update(cos=torch.cos(ang), sin=torch.sin(ang))
    elif op == "attention":
        lens, new = _lengths(case)
        bs = case["block"]
        pages = [-(-a // bs) for a in lens]
        blocks = sum(pages) + 2
        order = torch.randperm(blocks, generator=gen, device="cuda").int()
        p = torch.tensor(pages, device="cuda")
        col = torch.arange(max(pages), device="cuda")
        at = ((torch.cumsum(p, 0) - p)[:, None] + col).clamp(max=blocks - 1)
        rows = sum(new)
        s.update(cache=_random_cache(gen, blocks, case), table=torch.where(col < p[:, None], order[at], -1).int(),
                 lens=ints(lens), cu_rows=torch.cat((ints([0]), torch.cumsum(ints(new), 0).int())), blocks=blocks,
                 q=torch.randn(rows, case["heads"], case["dim"], generator=gen, device="cuda"),
                 out=torch.zeros(rows, case["heads"], case["dim"], device="cuda"))
    else:
        r, v = case["rows"], case["vocab"]
        x = torch.randn(r, v, generator=gen, device="cuda") * 2.2
        likely = torch.randint(0, v, (r, 3), generator=gen, device="cuda")
        x.scatter_add_(1, likely, 6 + 4 * torch.rand(r, 3, generator=gen, device="cuda"))
        if case["masked"]:  # every fourth row may give 3 to 40 tokens only
            keep = torch.rand(r, v, generator=gen, device="cuda") < 37.0 / v
            keep.scatter_(1, likely, True)
            limited = (torch.arange(r, device="cuda") % 4 == 1)[:, None]
            x = torch.where(keep | ~limited, x, -math.inf)
        other = torch.randint(0, v, (r,), generator=gen, device="cuda")
        ids = torch.where(torch.rand(r, generator=gen, device="cuda") < 0.7, likely[:, 0], other).int()
        s.update(logits=x, ids=ids)
    return s


# ----------------------------------------------------------------- one pass
_lib = None


def _nimf():
    """The framework's binding, bound to device 0."""
    global _lib
    if _lib is None:
        sys.path.insert(0, "nimformers-framework_b200")
        import nimf
        nimf.init(0)
        _lib = nimf
    return _lib


def _stream():
    return torch.cuda.current_stream().cuda_stream or 1  # 1: the legacy default stream


def run(s):
    op = s["case"]["op"]
    return {"reserve": _reserve, "append": _append, "attention": _attention, "logprobs": _logprobs}[op](s, s["case"])


def _cache_of(s, case):
    """The library's view of a pool, kept with the state as a program keeps it."""
    if "kv4" not in s:
        s["kv4"] = _nimf().KV4Cache(n_blocks=s["blocks"], n_kv_heads=case.get("kv_heads", 1), head_dim=case.get("dim", 64),
                                    block_size=case["block"], group=case.get("group", 32))
    return s["kv4"]


def _reserve(s, case):
    n, rows, bs = case["seqs"], s["rows"], case["block"]
    if own:
        lens = torch.empty_like(s["lens"])
        n_free, granted = torch.empty_like(s["n_free"]), torch.empty_like(s["lens"])
        cu = torch.empty(n + 1, dtype=torch.int32, device="cuda")
        slots, positions = (torch.empty(rows, dtype=torch.int32, device="cuda") for _ in range(2))
        _cache_of(s, case).reserve(n, case["width"], s["new"].data_ptr(), s["lens"].data_ptr(), lens.data_ptr(), s["table"].data_ptr(),
                                   s["free"].data_ptr(), s["n_free"].data_ptr(), n_free.data_ptr(), rows, cu.data_ptr(),
                                   slots.data_ptr(), positions.data_ptr(), granted.data_ptr(), stream=_stream())
        return dict(lens=lens, table=s["table"], n_free=n_free, cu_rows=cu, slots=slots, positions=positions, granted=granted)
    old, new = s["lens"].long(), s["new"].long()
    cu = torch.cat((torch.zeros_like(new[:1]), torch.cumsum(new, 0)))
    have, total = (old + bs - 1) // bs, (old + new + bs - 1) // bs
    fits = (total <= case["width"]) & (cu[1:] <= rows)
    need = torch.where(fits, total - have, 0)
    upto = torch.cumsum(need, 0)
    free = s["n_free"].long()
    granted = fits & ((need == 0) | (upto <= free))
    col = torch.arange(case["width"], device="cuda")
    fresh = granted[:, None] & (col >= have[:, None]) & (col < total[:, None])
    at = free - 1 - ((upto - need)[:, None] + col - have[:, None])
    table = torch.where(fresh, s["free"][at.clamp(0, s["free"].numel() - 1)], s["table"])
    t = torch.arange(rows, device="cuda")
    b = torch.searchsorted(cu[1:], t, right=True)
    live = b < n
    b = b.clamp(max=n - 1)
    pos = old[b] + t - cu[b]
    ok = live & granted[b]
    slot = table[b, (pos // bs).clamp(max=case["width"] - 1)].long() * bs + pos % bs
    return dict(lens=torch.where(granted, old + new, old).int(), table=table, n_free=(free - torch.where(granted, need, 0).sum()).int(), cu_rows=cu.int(),
                slots=torch.where(ok, slot, -1).int(), positions=torch.where(ok, pos, 0).int(), granted=granted.int())


def _rotate(x, cos, sin):
    h = x.shape[-1] // 2
    a, b, c, s = x[..., :h], x[..., h:], cos[:, None], sin[:, None]
    return torch.cat((a * c - b * s, a * s + b * c), -1)


def _append(s, case):
    if own:
        t = case["rows"]
        q, k, v = torch.empty_like(s["q"]), torch.empty_like(s["k"]), torch.empty_like(s["v"])
        kv4, st = _cache_of(s, case), _stream()
        kv4.append(s["cache"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), t, s["slots"].data_ptr(), q=s["q"].data_ptr(), q_out=q.data_ptr(),
                   n_heads=case["heads"], positions=s["positions"].data_ptr(), cos=s["cos"].data_ptr(), sin=s["sin"].data_ptr(),
                   max_seq=case["max_seq"], stream=st)
        kv4.read(s["cache"].data_ptr(), s["slots"].data_ptr(), t, k.data_ptr(), v.data_ptr(), stream=st)
        return dict(q=q, k=k, v=v)
    at = s["positions"].long()
    cos, sin = s["cos"][at], s["sin"][at]
    kept = (s["slots"] >= 0)[:, None, None]
    k = _value(*_code(_rotate(s["k"], cos, sin), case["group"]))
    v = _value(*_code(s["v"], case["group"]))
    return dict(q=_rotate(s["q"], cos, sin), k=torch.where(kept, k, 0.0), v=torch.where(kept, v, 0.0))


def _attention(s, case):
    n, h, kv, d = case["seqs"], case["heads"], case["kv_heads"], case["dim"]
    scale = 1.0 / math.sqrt(d)
    if own:
        kv4 = _cache_of(s, case)
        if "work" not in s:
            s["work"] = torch.empty(kv4.attention_workspace(h), dtype=torch.uint8, device="cuda")
        kv4.attention(s["cache"].data_ptr(), s["q"].data_ptr(), s["q"].shape[0], h, n, s["cu_rows"].data_ptr(), s["lens"].data_ptr(),
                      s["table"].data_ptr(), s["table"].shape[1], scale, s["out"].data_ptr(), s["work"].data_ptr(), s["work"].numel(),
                      max_new=case["prompt"], stream=_stream())
        return s["out"]
    width, most = s["table"].shape[1], case["prompt"]
    pages = s["cache"][s["table"].clamp(min=0).long()]  # [n, width, kv, block / 16, tile]
    k, v = _open(pages, d, case["group"])
    seq = width * case["block"]
    k = k.transpose(1, 2).reshape(n, kv, seq, d)
    v = v.transpose(1, 2).reshape(n, kv, seq, d)
    lens, cu = s["lens"].long(), s["cu_rows"].long()
    new = cu[1:] - cu[:-1]
    i = torch.arange(most, device="cuda")
    row = (cu[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].reshape(n, most, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(n, kv, h // kv * most, d)
    score = (q @ k.transpose(-1, -2)).mul_(scale).reshape(n, kv, h // kv, most, seq)
    last = lens[:, None] - new[:, None] + i
    seen = torch.arange(seq, device="cuda") <= torch.minimum(last, lens[:, None] - 1)[..., None]  # [n, most, seq]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    v = torch.where((torch.arange(seq, device="cuda") < lens[:, None])[:, None, :, None], v, 0.0)
    o = (p.reshape(n, kv, h // kv * most, seq) @ v).reshape(n, kv, h // kv, most, d) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, most, h, d)
    t = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted(cu[1:], t, right=True)
    live = (b < n)[:, None, None]
    b = b.clamp(max=n - 1)
    return torch.where(live, o[b, (t - cu[b]).clamp(0, most - 1)], s["out"])


def _logprobs(s, case):
    r, v, top = case["rows"], case["vocab"], case["top"]
    x = s["logits"]
    if own:
        f = lambda *shape: torch.empty(*shape, device="cuda")  # noqa: E731
        out = dict(logprob=f(r), entropy=f(r), rank=torch.empty(r, dtype=torch.int32, device="cuda"),
                   top_ids=torch.empty(r, top, dtype=torch.int32, device="cuda"), top_logprobs=f(r, top))
        _nimf().logprobs_dev(x.data_ptr(), r, v, s["ids"].data_ptr(), top, out["logprob"].data_ptr(), out["entropy"].data_ptr(),
                             out["rank"].data_ptr(), out["top_ids"].data_ptr(), out["top_logprobs"].data_ptr(), stream=_stream())
        return out
    m = x.amax(-1, keepdim=True)
    t = x - m
    e = t.exp()
    total = e.sum(-1)
    log_total = total.log()
    given = x.gather(1, s["ids"].long()[:, None])
    entropy = log_total - torch.where(e > 0, e * t, 0.0).sum(-1) / total
    ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top]
    return dict(logprob=t.gather(1, s["ids"].long()[:, None])[:, 0] - log_total, entropy=entropy, rank=((x > given).sum(-1) + 1).int(),
                top_ids=ids.int(), top_logprobs=t.gather(1, ids) - log_total[:, None])


# ------------------------------------------------------------ 64-bit answers
def _nibbles(rows, dim, key):
    """Codes [n, dim] of rows [n, dim / 2], each found by its place."""
    d = torch.arange(dim, device=rows.device)
    if key:
        word, nib = (d % 32 // 8) * (dim // 32) + d // 32, d % 8
    else:
        word, nib = (d % 32 // 4) * (dim // 64) + d // 64, d % 4 + 4 * (d % 64 // 32)
    return (rows[:, word * 4 + nib // 2].long() >> (4 * (nib % 2))) & 15


def exact(case, seed):
    op = case["op"]
    if op == "reserve":
        return None
    s = prepare(case, seed)
    if op == "append":
        # every step of the format is rounded to float32, so that its 64-bit
        # answer is each step computed in 64 bits and rounded
        r = lambda x: x.float().double()  # noqa: E731
        at = s["positions"].long()
        c, sn = s["cos"][at].double()[:, None], s["sin"][at].double()[:, None]
        h = case["dim"] // 2

        def turn(x):
            a, b = x.double()[..., :h], x.double()[..., h:]
            return torch.cat((r(r(a * c) - r(b * sn)), r(r(a * sn) + r(b * c))), -1)

        def held(x):
            g = x.unflatten(-1, (-1, case["group"]))
            low = g.amin(-1, keepdim=True)
            step = r(r(g.amax(-1, keepdim=True) - low) / 15)
            code = torch.where(step > 0, torch.round(r(r(g - low) / step)), 0.0).clamp(max=15)
            return torch.where((s["slots"] < 0)[:, None, None], 0.0, r(r(code * step) + low).flatten(-2))

        return dict(q=turn(s["q"]), k=held(turn(s["k"])), v=held(s["v"].double()))
    if op == "logprobs":
        x = s["logits"].double()
        lse = torch.logsumexp(x, -1)
        logp = x - lse[:, None]
        p = logp.exp()
        ids = torch.sort(s["logits"], dim=-1, descending=True, stable=True)[1][:, :case["top"]]
        return dict(logprob=logp.gather(1, s["ids"].long()[:, None])[:, 0], entropy=-torch.where(p > 0, p * logp, 0.0).sum(-1),
                    rank=None, top_ids=None, top_logprobs=logp.gather(1, ids))
    lens, new = _lengths(case)
    h, kv, d, group, bs = case["heads"], case["kv_heads"], case["dim"], case["group"], case["block"]
    half, par = TILE * d // 2, TILE * 8 * (d // group)
    out = torch.zeros(sum(new), h, d, dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        for head in range(kv):
            tiles = s["cache"][s["table"][b, :-(-n // bs)].long(), head].reshape(-1, _tile_bytes(case))
            got = []
            for key, codes, at in ((True, 0, 2 * half), (False, half, 2 * half + par)):
                c = _nibbles(tiles[:, codes:codes + half].reshape(-1, d // 2), d, key)[:n].double()
                p = tiles[:, at:at + par].contiguous().view(torch.float32).reshape(-1, d // group, TILE, 2)
                p = p.permute(0, 2, 1, 3).reshape(-1, d // group, 2)[:n].double().repeat_interleave(group, 1)
                got.append(c * p[..., 0] + p[..., 1])
            q = s["q"][row:row + m, head * (h // kv):(head + 1) * (h // kv)].double()
            a = torch.einsum("ihd,jd->hij", q, got[0]) / math.sqrt(d)
            hidden = torch.arange(n, device="cuda") > n - m + torch.arange(m, device="cuda")[:, None]
            a = torch.softmax(a.masked_fill(hidden, -math.inf), -1)
            out[row:row + m, head * (h // kv):(head + 1) * (h // kv)] = torch.einsum("hij,jd->ihd", a, got[1])
        row += m
    return out
