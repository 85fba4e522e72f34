"""Token generation's operators, as measured cases: keys and values appended to a paged cache held in 4 bits (with
the position rotation on the way), the cache read back, attention over it, and the adjustment of logits before a
token is drawn from them.

Each case has a plain form in elementary torch operations in 32 bits (``own`` false) and the framework's call
(``own`` true).  Both take the same state: tensors in the layouts that ``scratchtape_b200.kv4`` documents.

The cache's layout, restated: ``data`` is uint8 [pages, kv_heads, page / 16, tile], a tile being 16 tokens of one
head.  With d channels, groups of G channels and d / G groups, a tile holds
  8 d bytes    key codes [group][token][G / 2], channel 2 b of the group in the low half of byte b;
  8 d bytes    value codes [d / 2][16], channel 2 p in the low half of row p; token t stands in column ORDER[t];
  64 d/G bytes key (scale, zero) [group][token] in float16, then the same for the values;
a code c stands for c * scale + zero.  Slot s is token s % 16 of tile (s % page) / 16 of page s / page.
"""
import math

import torch

own = False

ORDER = [4 * ((t & 7) >> 1) + 2 * (t & 1) + (t >> 3) for t in range(16)]
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _spread(lo, hi, n, salt=0):
    """n whole numbers over lo..hi, the largest first, the same ones for the same arguments."""
    return [hi] + [lo + ((i + salt) * 40503 * 65537 % 65521) * (hi - lo) // 65520 for i in range(1, n)]


def listed():
    return [
        # the byte-level model's own shape (4 heads of 64, float32, learned positions): one token for each of a few
        # sequences, where the call's latency is all there is
        dict(name="append 4 tokens f32", op="append", batch=4, new_lo=1, new=1, context=9, kv_heads=4, heads=4, d=64,
             group=64, page=16, rotary=0, interleaved=False, type="f32"),
        # one decoding step of a busy server: a token for each of 128 sequences
        dict(name="append 128 tokens bf16", op="append", batch=128, new_lo=1, new=1, context=13, kv_heads=8, heads=32,
             d=128, group=64, page=16, rotary=128, interleaved=False, type="bf16"),
        # prompts of odd lengths taken in at once, after contexts that end inside a tile
        dict(name="append prompts 8k bf16", op="append", batch=6, new_lo=403, new=2048, context=1001, kv_heads=8,
             heads=32, d=128, group=64, page=64, rotary=128, interleaved=False, type="bf16"),
        # a short sequence moved out of the cache
        dict(name="read 1000 f16", op="read", tokens=1000, kv_heads=4, d=64, group=32, page=16, type="f16"),
        # the whole of a long context moved out of it
        dict(name="read 64k bf16", op="read", tokens=65536, kv_heads=8, d=128, group=64, page=64, type="bf16"),
        # the byte-level model answering: four sequences, a query each
        dict(name="attend 4 x 128 f32", op="attend", batch=4, q_lo=1, q=1, kv_lo=60, kv=128, kv_heads=4, heads=4,
             d=64, group=64, page=16, causal=True, window=0, one=True, lse=True, type="f32"),
        # an ordinary decoding step with shared heads and ragged contexts
        dict(name="attend 32 x 4k bf16", op="attend", batch=32, q_lo=1, q=1, kv_lo=500, kv=4096, kv_heads=8, heads=32,
             d=128, group=64, page=64, causal=True, window=0, one=False, lse=False, type="bf16"),
        # one sequence with a very long context
        dict(name="attend 1 x 128k f16", op="attend", batch=1, q_lo=1, q=1, kv_lo=131000, kv=131000, kv_heads=8,
             heads=32, d=128, group=64, page=128, causal=True, window=0, one=False, lse=True, type="f16"),
        # the largest decoding step: the cache takes gigabytes
        dict(name="attend 64 x 16k bf16", op="attend", batch=64, q_lo=1, q=1, kv_lo=15000, kv=16384, kv_heads=8,
             heads=64, d=128, group=64, page=64, causal=True, window=0, one=False, lse=False, type="bf16"),
        # pieces of prompts attending to all that came before them
        dict(name="attend 2k rows 8k bf16", op="attend", batch=3, q_lo=300, q=1024, kv_lo=2000, kv=8192, kv_heads=8,
             heads=32, d=128, group=64, page=64, causal=True, window=0, one=False, lse=False, type="bf16"),
        # the byte-level model's vocabulary
        dict(name="logits 4 x 256 f32", op="logits", rows=4, vocab=256, history=128, bias=3, masks=2, type="f32"),
        # a large batch over a large vocabulary, most rows under a grammar
        dict(name="logits 256 x 128k bf16", op="logits", rows=256, vocab=131075, history=4096, bias=64, masks=200,
             type="bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append", "read", "attend", "attend", "attend", "logits"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "logits":
        rows = log(1, 256)
        vocab = log(200, min(131072, 256 * 131072 // rows))
        return dict(op=op, rows=rows, vocab=vocab, history=log(1, 4096), bias=rng.choice([0, log(1, 64)]),
                    masks=rng.choice([0, log(1, rows + 1)]), type=kind)
    d = rng.choice([64, 128, 128])
    group = rng.choice([g for g in (32, 64, 64, 128) if g <= d])
    page = rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8, 8])
    common = dict(kv_heads=kv_heads, d=d, group=group, page=page, type=kind)
    if op == "read":
        return dict(op=op, tokens=log(1, 65536), **common)
    if op == "append":
        batch = log(1, 128)
        new = 1 if rng.random() < 0.4 else log(1, max(2, 3500 // batch))
        return dict(op=op, batch=batch, new_lo=rng.randint((new + 1) // 2, new), new=new, context=rng.randint(0, 60),
                    heads=heads, rotary=rng.choice([0, d, d, d // 2]), interleaved=rng.random() < 0.3, **common)
    batch = log(1, 64)
    if rng.random() < 0.65:  # single tokens, or a few that were guessed ahead
        q = rng.choice([1, 1, 1, rng.randint(2, 8)])
        kv = log(1, max(2, min(131072, 1000000 // (batch * q))))
    else:
        batch = min(batch, 6)
        q = log(9, 1024 // batch)
        kv = max(q, log(64, 8192))
    return dict(op=op, batch=batch, q_lo=rng.randint(1, q), q=q, kv_lo=rng.randint(0, kv), kv=kv, heads=heads,
                causal=rng.random() < 0.8, window=rng.choice([0, 0, 0, log(1, 4096)]), one=rng.random() < 0.25,
                lse=rng.random() < 0.5, **common)


# ---- the cases' sizes and inputs -------------------------------------------------------------------------------


def _tile_bytes(d, group):
    return 16 * d + 128 * (d // group)


def _lengths(case):
    """append: (tokens before, tokens new) of each sequence; attend: (keys, queries) of each."""
    n = case["batch"]
    if case["op"] == "append":
        return [case["context"] * (i % 3) // 2 for i in range(n)], _spread(case["new_lo"], case["new"], n)
    return _spread(case["kv_lo"], case["kv"], n), _spread(case["q_lo"], case["q"], n, 7)


def _pages(case):
    """Pages of each sequence."""
    if case["op"] == "append":
        lens = [a + b for a, b in zip(*_lengths(case))]
    elif case["op"] == "read":
        lens = [case["tokens"]]
    else:
        lens = _lengths(case)[0]
    return [-(-x // case["page"]) for x in lens]


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _quantise(x, group):
    """x [..., d] -> whole codes [..., d], scale and zero [..., d / group] in float16."""
    x = torch.nan_to_num(x, nan=0.0, posinf=65504.0, neginf=-65504.0).clamp(-65504.0, 65504.0)
    g = x.unflatten(-1, (-1, group))
    zero = g.amin(-1).to(torch.float16)
    scale = ((g.amax(-1) - zero.float()) / 15.0).to(torch.float16)
    s = scale.float()
    inverse = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    code = torch.round((g - zero.float()[..., None]) * inverse[..., None]).clamp(0.0, 15.0)
    return code.flatten(-2).to(torch.uint8), scale, zero


def _pack(k, v, group):
    """Rotated keys and values [tiles, 16, d] in 32 bits -> tiles uint8 [tiles, tile bytes]."""
    n, _, d = k.shape
    kc, ks, kz = _quantise(k, group)
    vc, vs, vz = _quantise(v, group)
    half = lambda c: c[..., 0::2] | (c[..., 1::2] << 4)  # noqa: E731
    kb = half(kc).view(n, 16, d // group, group // 2).transpose(1, 2).reshape(n, -1)
    order = torch.tensor(ORDER, device=k.device)
    vb = torch.empty((n, d // 2, 16), dtype=torch.uint8, device=k.device)
    vb[:, :, order] = half(vc).transpose(1, 2)
    meta = [torch.stack([s, z], -1).transpose(1, 2).contiguous().view(torch.uint8).view(n, -1)
            for s, z in ((ks, kz), (vs, vz))]
    return torch.cat([kb, vb.view(n, -1)] + meta, 1)


def _unpack(data, d, group):
    """data [..., tile bytes] -> keys, values [..., 16, d] in 32 bits."""
    lead, ng = data.shape[:-1], d // group
    both = lambda b: torch.stack([b & 15, b >> 4], -1).flatten(-2)  # noqa: E731
    kc = both(data[..., : 8 * d].reshape(*lead, ng, 16, group // 2)).transpose(-2, -3)
    order = torch.tensor(ORDER, device=data.device)
    vb = data[..., 8 * d: 16 * d].reshape(*lead, d // 2, 16)[..., order].transpose(-1, -2)
    vc = both(vb).unflatten(-1, (ng, group))
    out = []
    for c, at in ((kc, 16 * d), (vc, 16 * d + 64 * ng)):
        meta = data[..., at: at + 64 * ng].contiguous().view(torch.float16).reshape(*lead, ng, 16, 2)
        meta = meta.transpose(-2, -3).float()
        out.append((c.float() * meta[..., :1] + meta[..., 1:]).flatten(-2))
    return out


def _slots(data, d, group):
    """Every slot's keys and values [slots, heads, d] in 32 bits."""
    return [x.permute(0, 2, 3, 1, 4).flatten(0, 2) for x in _unpack(data, d, group)]


def _cache(case, gen, total):
    """A cache of `total` pages full of keys (a few channels larger and off centre, as rotated keys have them) and
    values."""
    d, group, heads, tiles = case["d"], case["group"], case["kv_heads"], case["page"] // 16
    data = torch.empty((total, heads, tiles, _tile_bytes(d, group)), dtype=torch.uint8, device="cuda")
    at = torch.rand((heads, 1, 1, d), generator=gen, device="cuda")
    gain, shift = 1.0 + 2.0 * (at > 0.94), 1.5 * (at > 0.9)
    step = max(1, (1 << 27) // (heads * case["page"] * d))
    for i in range(0, total, step):
        n = min(step, total - i)
        k = _randn(gen, n, heads, tiles, 16, d) * gain[None] + shift[None]
        v = _randn(gen, n, heads, tiles, 16, d)
        data[i: i + n] = _pack(k.view(-1, 16, d), v.view(-1, 16, d), group).view(n, heads, tiles, -1)
    return data


def _table(case, gen):
    """(pages of the cache, page numbers of each sequence int32 [batch, most], the rest out of use)."""
    need = _pages(case)
    total = sum(need) + 2
    numbers = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    most = max(1, max(need))
    ends = torch.tensor(need, device="cuda").cumsum(0)
    at = torch.arange(most, device="cuda")[None] + (ends - torch.tensor(need, device="cuda"))[:, None]
    return total, torch.where(at < ends[:, None], numbers[at.clamp(max=total - 1)], -1).contiguous()


def _rotation(case):
    """cos and sin [positions, rotary / 2]."""
    half = case["rotary"] // 2
    rate = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / max(1, half))
    angle = torch.arange(8192, dtype=torch.float64, device="cuda")[:, None] * rate
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]
    ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device="cuda")  # noqa: E731
    s = dict(case)
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = (_randn(gen, rows, vocab) * 3.0).to(kind)
        length = _spread(case["history"] // 4, case["history"], rows)
        s["starts"] = torch.cat([ints([0]), ints(length).cumsum(0).to(torch.int32)])
        # tokens repeat as they do in text: small numbers often, large ones rarely; a few are padding
        u = torch.rand(sum(length), generator=gen, device="cuda")
        s["tokens"] = torch.where(u > 0.995, -1, (vocab * u ** 3).to(torch.int32)).to(torch.int32)
        s["prompt"] = ints([x * (i % 4) // 4 for i, x in enumerate(length)])
        one = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, generator=gen, device="cuda")  # noqa: E731
        s["repetition"], s["presence"], s["frequency"] = one(1.0, 1.3), one(-0.5, 1.0), one(0.0, 0.3)
        if case["bias"]:
            counts = _spread(0, case["bias"], rows, 3)
            s["bias_starts"] = torch.cat([ints([0]), ints(counts).cumsum(0).to(torch.int32)])
            n = sum(counts)
            s["bias_tokens"] = torch.randint(0, vocab, (n,), generator=gen, device="cuda", dtype=torch.int32)
            s["bias_values"] = _randn(gen, n) * 5.0
        if case["masks"]:
            words = -(-vocab // 32)
            mask = torch.randint(-2 ** 31, 2 ** 31, (case["masks"], words), generator=gen, device="cuda",
                                 dtype=torch.int64)
            s["mask"] = (mask & torch.randint(-2 ** 31, 2 ** 31, mask.shape, generator=gen, device="cuda",
                                              dtype=torch.int64)).to(torch.int32)
            s["mask_rows"] = ints([i % case["masks"] if i % 5 else -1 for i in range(rows)])
        return s
    if case["op"] == "read":
        total, table = _table(case, gen)
        s["data"] = _cache(case, gen, total)
        i = torch.arange(case["tokens"], device="cuda")
        s["slots"] = table[0].long()[i // case["page"]] * case["page"] + i % case["page"]
        return s
    total, table = _table(case, gen)
    s["data"], s["pages"] = _cache(case, gen, total), table
    before, new = _lengths(case)
    if case["op"] == "append":
        n = sum(new)
        q, k, v = (_randn(gen, n, h, case["d"]).to(kind) for h in (case["heads"], case["kv_heads"], case["kv_heads"]))
        s.update(q=q, k=k, v=v)
        ends = ints(new, torch.int64).cumsum(0)
        i = torch.arange(n, device="cuda")
        row = torch.searchsorted(ends, i, right=True)
        pos = ints(before, torch.int64)[row] + i - (ends - ints(new, torch.int64))[row]
        s["slots"] = table[row, pos // case["page"]].long() * case["page"] + pos % case["page"]
        if n > 16:  # places that a batch of fixed size leaves empty
            s["slots"][torch.randint(0, n, (n // 50,), generator=gen, device="cuda")] = -1
        s["positions"] = pos.to(torch.int32)
        s["cos"], s["sin"] = _rotation(case) if case["rotary"] else (None, None)
        s["every"] = torch.arange(total * case["page"], device="cuda")
        return s
    s["kv_len"], s["max_q"] = ints(before), max(new)
    n = sum(new)
    s["q"] = (_randn(gen, n, case["heads"], case["d"]) * 1.5).to(kind)
    s["q_start"] = torch.cat([ints([0]), ints(new).cumsum(0).to(torch.int32)])
    s["scale"] = case["d"] ** -0.5
    return s


# ---- one pass --------------------------------------------------------------------------------------------------


def run(s):
    if own:
        return _own(s)
    return {"append": _append, "read": _read, "attend": _attend, "logits": _logits}[s["op"]](s)


def _own(s):
    if s["op"] == "logits":
        from scratchtape_b200 import logits
        bias = (s["bias_tokens"], s["bias_values"], s["bias_starts"]) if s["bias"] else None
        mask = (s["mask"], s["mask_rows"]) if s["masks"] else None
        return logits.adjust(s["logits"], s["tokens"], s["starts"], s["prompt"], s["repetition"], s["presence"],
                             s["frequency"], bias=bias, mask=mask)
    from scratchtape_b200 import kv4
    if s["op"] == "read":
        return kv4.read(s["data"], s["slots"], s["d"], s["group"], TYPES[s["type"]])
    if s["op"] == "append":
        q = kv4.append(s["data"], s["k"], s["v"], s["slots"], s["group"], q=s["q"] if s["rotary"] else None,
                       cos=s["cos"], sin=s["sin"], positions=s["positions"], interleaved=s["interleaved"])
        k, v = kv4.read(s["data"], s["every"], s["d"], s["group"], TYPES[s["type"]])
        return (q, k, v) if s["rotary"] else (k, v)
    return kv4.attend(s["q"], s["data"], s["pages"], s["kv_len"], s["scale"], s["group"], q_start=s["q_start"],
                      max_q=s["max_q"], causal=s["causal"], one=s["one"], window=s["window"], return_lse=s["lse"])


def _rotate(x, s):
    """x [n, heads, d] in 32 bits, its first `rotary` channels turned by the token's position."""
    r = s["rotary"]
    if not r:
        return x
    cos, sin = (t[s["positions"].long()][:, None] for t in (s["cos"], s["sin"]))
    turned, rest = x[..., :r], x[..., r:]
    if s["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., : r // 2], turned[..., r // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _append(s):
    kind, d, group, page = TYPES[s["type"]], s["d"], s["group"], s["page"]
    ng, ok = d // group, s["slots"] >= 0
    slot = s["slots"][ok]
    k, v = _rotate(s["k"].float(), s)[ok], s["v"].float()[ok]
    kc, ks, kz = _quantise(k, group)
    vc, vs, vz = _quantise(v, group)
    p, t, r = slot // page, slot % page // 16, slot % 16
    data = s["data"]
    ends = [8 * d, 16 * d, 16 * d + 64 * ng, 16 * d + 128 * ng]
    kb, vb, km, vm = (data[..., a:b] for a, b in zip([0] + ends, ends))
    half = lambda c: c[..., 0::2] | (c[..., 1::2] << 4)  # noqa: E731
    kb = kb.unflatten(-1, (ng, 16, group // 2))
    kb[p, :, t, :, r] = half(kc).unflatten(-1, (ng, group // 2))
    vb.unflatten(-1, (d // 2, 16))[p, :, t, :, torch.tensor(ORDER, device=r.device)[r]] = half(vc)
    for m, a, b in ((km, ks, kz), (vm, vs, vz)):
        pair = torch.stack([a, b], -1).view(torch.uint8)  # [n, heads, groups, 4 bytes]
        m.unflatten(-1, (ng, 16, 4))[p, :, t, :, r] = pair.view(*a.shape, 4)
    k, v = _slots(data, d, group)
    q = _rotate(s["q"].float(), s).to(kind)
    k, v = k.to(kind), v.to(kind)
    return (q, k, v) if s["rotary"] else (k, v)


def _read(s):
    k, v = _slots(s["data"], s["d"], s["group"])
    return k[s["slots"]].to(TYPES[s["type"]]), v[s["slots"]].to(TYPES[s["type"]])


def _attend(s):
    d, heads, kv_heads, page = s["d"], s["heads"], s["kv_heads"], s["page"]
    batch, n = s["batch"], s["q"].shape[0]
    start, length = s["q_start"].long(), s["kv_len"].long()
    count = start[1:] - start[:-1]
    every = torch.arange(n, device=start.device)
    row = torch.searchsorted(start[1:], every, right=True)
    most = s["pages"].shape[1]
    k, v = _unpack(s["data"][s["pages"].long().clamp(min=0)], d, s["group"])
    k, v = (x.transpose(1, 2).flatten(2, 4) for x in (k, v))  # [batch, kv head, key, d]
    q = torch.zeros((batch, s["max_q"], heads, d), device=start.device)
    q[row, every - start[row]] = s["q"].float()
    q = q.view(batch, s["max_q"], kv_heads, heads // kv_heads, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    x = (q @ k.transpose(-1, -2)).mul_(s["scale"])  # [batch, kv head, shared head and query, key]
    x = x.view(batch, kv_heads, heads // kv_heads, s["max_q"], most * page)
    key = torch.arange(most * page, device=start.device)
    at = length[:, None] - count[:, None] + torch.arange(s["max_q"], device=start.device)  # each query's position
    seen = (key < length[:, None])[:, None]
    if s["causal"]:
        seen = seen & (key <= at[..., None])
    if s["window"]:
        seen = seen & (key > at[..., None] - s["window"])
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    if s["one"]:
        top = top.clamp(min=0.0)
    x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    if s["one"]:
        total = total + torch.exp(-top)
    lse = (torch.log(total) + top)[..., 0]
    o = (x.flatten(2, 3) @ v).unflatten(2, (-1, s["max_q"])) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[row, every - start[row]].to(TYPES[s["type"]])
    lse = lse.permute(0, 3, 1, 2).flatten(2, 3)[row, every - start[row]]
    return (o, lse) if s["lse"] else o


def _logits(s):
    rows, vocab = s["rows"], s["vocab"]
    x = s["logits"].float()
    i = torch.arange(s["tokens"].numel(), device=x.device)
    row = torch.searchsorted(s["starts"][1:].long(), i, right=True)
    real = (s["tokens"] >= 0) & (s["tokens"] < vocab)
    flat = row * vocab + s["tokens"]
    answer = i - s["starts"].long()[row] >= s["prompt"].long()[row]
    ones = torch.ones((), dtype=torch.int32, device=x.device)
    met, said = (torch.zeros(rows * vocab, dtype=torch.int32, device=x.device) for _ in range(2))
    met.index_put_((flat[real],), ones, accumulate=True)
    said.index_put_((flat[real & answer],), ones, accumulate=True)
    met, said = met.view(rows, vocab), said.view(rows, vocab)
    rep = s["repetition"][:, None]
    x = torch.where(met > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * said - s["presence"][:, None] * (said > 0)
    if s["bias"]:
        j = torch.arange(s["bias_tokens"].numel(), device=x.device)
        at = torch.searchsorted(s["bias_starts"][1:].long(), j, right=True)
        x = x.index_put((at, s["bias_tokens"].long()), s["bias_values"], accumulate=True)
    if s["masks"]:
        bit = torch.arange(vocab, device=x.device)
        free = (s["mask_rows"] < 0)[:, None]
        word = s["mask"][s["mask_rows"].long().clamp(min=0)][:, bit // 32]
        x = torch.where(free | ((word >> (bit % 32)) & 1 > 0), x, -math.inf)
    return x.to(TYPES[s["type"]])


# ---- what a pass cannot do without -----------------------------------------------------------------------------


def _seen_pairs(case):
    pairs = 0
    for keys, queries in zip(*_lengths(case)):
        for i in range(queries):
            at = keys - queries + i
            hi = min(keys, at + 1) if case["causal"] else keys
            lo = max(0, at - case["window"] + 1) if case["window"] else 0
            pairs += max(0, hi - lo)
    return pairs


def work(case):
    size = SIZE[case["type"]]
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        history = sum(_spread(case["history"] // 4, case["history"], rows))
        masked = min(rows, case["masks"]) * -(-vocab // 32) * 4 if case["masks"] else 0
        return {"bytes": 2 * rows * vocab * size + 4 * history + masked + 8 * rows * case["bias"] // 2, "flops": 0}
    d, heads = case["d"], case["kv_heads"]
    token = heads * (d + 8 * (d // case["group"]))  # bytes of one token's keys and values in the cache
    if case["op"] == "read":
        return {"bytes": case["tokens"] * (token + 8 + 2 * heads * d * size), "flops": 4 * case["tokens"] * heads * d}
    if case["op"] == "append":
        n, whole = sum(_lengths(case)[1]), (sum(_pages(case)) + 2) * case["page"]
        turned = n * 2 * case["heads"] * d * size if case["rotary"] else 0
        return {"bytes": n * (2 * heads * d * size + token + 8) + turned + whole * (token + 2 * heads * d * size),
                "flops": 10 * n * heads * d}
    keys, queries = _lengths(case)
    # the keys that some query of the sequence sees
    used = sum(min(k, max(0, q + case["window"] - 1)) if case["window"] else k for k, q in zip(keys, queries))
    flops = 4 * case["heads"] * d * _seen_pairs(case)
    return {"bytes": used * token + 2 * sum(queries) * case["heads"] * d * size, "flops": flops}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------


def _values64(data, d, group):
    """Every slot's keys and values [slots, heads, d] in 64 bits, by the address of each code."""
    pages, heads, tiles, tile = data.shape
    by_tile = data.permute(0, 2, 1, 3).reshape(pages * tiles, heads, tile)
    ng, dev = d // group, data.device
    t, c = torch.arange(16, device=dev)[:, None], torch.arange(d, device=dev)[None]
    key_at = (c // group) * (8 * group) + t * (group // 2) + c % group // 2
    value_at = 8 * d + c // 2 * 16 + 4 * (t % 8 // 2) + 2 * (t % 2) + t // 8
    out = []
    for at, meta in ((key_at, 16 * d), (value_at, 16 * d + 64 * ng)):
        byte = by_tile[:, :, at].long()
        code = torch.where((c % 2 == 1).expand_as(at), byte // 16, byte % 16).double()
        where = meta + ((c // group) * 16 + t) * 4
        scale, zero = (torch.stack([by_tile[:, :, where + o], by_tile[:, :, where + o + 1]], -1).view(torch.float16)
                       [..., 0].double() for o in (0, 2))
        out.append((code * scale + zero).permute(0, 2, 1, 3).reshape(-1, heads, d))
    return out


def _quantised64(x, group):
    n, heads, d = x.shape
    g = x.view(n, heads, d // group, group).clamp(-65504.0, 65504.0)
    zero = g.min(-1, keepdim=True).values.half().double()
    scale = ((g.max(-1, keepdim=True).values - zero) / 15).half().double()
    return (torch.where(scale > 0, torch.round((g - zero) / scale.clamp(min=1e-30)), 0.0).clamp(0, 15) * scale
            + zero).view(n, heads, d)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logits":
        return _logits64(s)
    d, group = case["d"], case["group"]
    if case["op"] == "read":
        used = s["slots"] // case["page"]
        numbers, back = torch.unique(used, return_inverse=True)
        k, v = _values64(s["data"][numbers], d, group)
        at = back * case["page"] + s["slots"] % case["page"]
        return k[at], v[at]
    if case["op"] == "append":
        r = case["rotary"]

        def turn(x):
            x = x.double()
            if not r:
                return x
            first = torch.arange(0, r, 2) if case["interleaved"] else torch.arange(r // 2)
            second = first + 1 if case["interleaved"] else first + r // 2
            angle = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None]
            z = torch.complex(x[..., first], x[..., second]) * angle
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            return y

        k, v = _values64(s["data"], d, group)
        real = torch.nonzero(s["slots"] >= 0)[:, 0]
        k[s["slots"][real]] = _quantised64(turn(s["k"])[real], group)
        v[s["slots"][real]] = _quantised64(s["v"].double()[real], group)
        return (turn(s["q"]), k, v) if r else (k, v)
    keys, queries = _lengths(case)
    if sum(k * q for k, q in zip(keys, queries)) * case["heads"] > 1 << 31:
        return None
    share, page = case["heads"] // case["kv_heads"], case["page"]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    begin = 0
    for b, (m, n) in enumerate(zip(keys, queries)):
        rows = slice(begin, begin + n)
        begin += n
        if case["one"]:
            lse[rows] = 0.0
        if not m:
            continue
        k, v = (x[:m].transpose(0, 1) for x in _values64(s["data"][s["pages"][b, : -(-m // page)].long()], d, group))
        pos = torch.arange(m - n, m, device="cuda")[:, None]
        key = torch.arange(m, device="cuda")[None]
        hidden = torch.zeros((n, m), dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden |= key > pos
        if case["window"]:
            hidden |= pos - key >= case["window"]
        for h in range(case["heads"]):
            x = (s["q"][rows, h].double() @ k[h // share].T) * s["scale"]
            x[hidden] = -math.inf
            e = torch.cat([x, torch.zeros((n, 1), dtype=x.dtype, device="cuda")], 1) if case["one"] else x
            lse[rows, h] = torch.logsumexp(e, 1)
            some = lse[rows, h] > -math.inf
            p = torch.exp(x - torch.where(some, lse[rows, h], 0.0)[:, None])
            o[rows, h] = p @ v[h // share]
    return (o, lse) if case["lse"] else o


def _logits64(s):
    x = s["logits"].double()
    if s["rows"] * s["vocab"] > 1 << 26:
        return None
    starts, prompt = s["starts"].tolist(), s["prompt"].tolist()
    bias = s["bias_starts"].tolist() if s["bias"] else None
    for r in range(s["rows"]):
        told = s["tokens"][starts[r]: starts[r + 1]].long()
        said = told[prompt[r]:]
        told, said = (t[(t >= 0) & (t < s["vocab"])] for t in (told, said))
        seen, rep = told.unique(), s["repetition"][r].double()
        x[r, seen] = torch.where(x[r, seen] > 0, x[r, seen] / rep, x[r, seen] * rep)
        which, times = said.unique(return_counts=True)
        x[r, which] -= s["presence"][r].double() + s["frequency"][r].double() * times
        if s["bias"]:
            part = slice(bias[r], bias[r + 1])
            x[r].index_add_(0, s["bias_tokens"][part].long(), s["bias_values"][part].double())
        if s["masks"] and (m := int(s["mask_rows"][r])) >= 0:
            bits = s["mask"][m][:, None] >> torch.arange(32, device=x.device, dtype=torch.int32) & 1
            x[r][bits.flatten()[: s["vocab"]] == 0] = -math.inf
    return x
