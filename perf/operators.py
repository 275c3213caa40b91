"""The operators for serving with drafted tokens: rotary positions with the cache rows they go to, rows read back from a cache,
attention of a tree of drafted tokens over a paged cache, and penalties, biases and grammar masks on logits.

A case names its operator (`op`).  Caches are paged like the engines': pages of 64 rows per KV head, rows of 128 values whose
16-byte pieces lie at index (piece XOR (row mod 8)), bf16, or e4m3 codes with one fp32 scale per row.  Head counts are those of
the repository's 8B (32 / 8) and mixture-of-experts (32 / 4) shapes and of its tests.  The sequences of a batch have lengths
between half of `ctx` and `ctx`.
"""
import math
import random

import torch

own = False

BF16, F8 = torch.bfloat16, torch.float8_e4m3fn
PAGE, D = 64, 128
DEV = "cuda:0"
E4M3_MAX = 448.0


def _append(batch, tokens, heads, kv, ctx, kind, layout, rot, norm, name=None):
    c = dict(op="append", batch=batch, tokens=tokens, heads=heads, kv=kv, ctx=ctx, kind=kind, layout=layout, rot=rot, norm=norm)
    return dict(c, name=name) if name else c


def _read(batch, kv, ctx, kind, name=None):
    c = dict(op="read", batch=batch, kv=kv, ctx=ctx, kind=kind)
    return dict(c, name=name) if name else c


def _attend(batch, tokens, heads, kv, ctx, kind, name=None):
    c = dict(op="attend", batch=batch, tokens=tokens, heads=heads, kv=kv, ctx=ctx, kind=kind)
    return dict(c, name=name) if name else c


def _logits(requests, tokens, vocab, history, kind, bias, grammar, name=None):
    c = dict(op="logits", requests=requests, tokens=tokens, vocab=vocab, history=history, kind=kind, bias=bias, grammar=grammar)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token of one sequence into an e4m3 cache: launch latency
        _append(1, 1, 32, 8, 333, "e4m3", "half", 128, False, name="append_token"),
        # trees of 16 drafted tokens of a serving batch, half of each head rotated in pairs, bf16 cache
        _append(32, 16, 32, 8, 1500, "bf16", "interleaved", 64, False, name="append_trees"),
        # two long prompts with q/k norms going into a quantised cache
        _append(2, 4096, 32, 4, 4096, "e4m3", "half", 128, True, name="append_prompts"),
        # a short conversation handed back to a program that wants bf16 rows
        _read(1, 8, 333, "e4m3", name="read_short"),
        # a batch of long sequences read back whole
        _read(16, 8, 4131, "e4m3", name="read_batch"),
        # one token of one short sequence: launch latency
        _attend(1, 1, 32, 8, 333, "bf16", name="attend_token"),
        # a serving batch, one token each
        _attend(64, 1, 32, 8, 2112, "e4m3", name="attend_batch"),
        # trees of 16 drafted tokens over quantised caches, ragged
        _attend(8, 16, 32, 8, 4131, "e4m3", name="attend_trees"),
        # large trees of a model with eight query heads per KV head: arithmetic counts as much as bytes
        _attend(4, 63, 32, 4, 2050, "bf16", name="attend_large_trees"),
        # a chain of eight drafted tokens behind a very long context
        _attend(1, 8, 32, 8, 131000, "e4m3", name="attend_long"),
        # one row of an 8B vocabulary with the penalties of a chat
        _logits(1, 1, 128256, 2112, "bf16", 0, False, name="logits_row"),
        # the rows of 64 trees, with biases and a grammar mask per row
        _logits(64, 8, 151936, 4096, "bf16", 32, True, name="logits_trees"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "logits"])
    heads, kv = rng.choice([(32, 8), (32, 4), (8, 2), (8, 1)])
    kind = rng.choice(["bf16", "e4m3"])
    if op == "append":
        tokens = _log(rng, 1, 4096)
        return _append(_log(rng, 1, 64), tokens, heads, kv, max(tokens, _log(rng, 1, 8192)), kind, rng.choice(["half", "interleaved"]),
                       rng.choice([32, 64, 96, 128]), rng.random() < 0.5)
    if op == "read":
        return _read(_log(rng, 1, 64), kv, _log(rng, 1, 16384), kind)
    if op == "attend":
        return _attend(_log(rng, 1, 64), _log(rng, 1, 64), heads, kv, _log(rng, 1, 131000), kind)
    return _logits(_log(rng, 1, 64), _log(rng, 1, 16), _log(rng, 2000, 151936), _log(rng, 1, 8192), rng.choice(["bf16", "fp32"]),
                   rng.choice([0, 1, 7, 64]), rng.random() < 0.5)


def draw(rng):
    """A case of the same ranges that moves at most 256 MB and computes at most 64 GFLOP."""
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= 256e6 and w["flops"] <= 64e9 and (c["op"] != "append" or c["batch"] * c["ctx"] <= 65536):
            return c


def _lengths(case):
    """Rows that the sequences hold: from half of ctx to ctx, evenly."""
    n, top = case["batch"], case["ctx"]
    return [top - (top // 2) * i // max(1, n - 1) for i in range(n)]


def _row_bytes(kind):
    return 2 * D if kind == "bf16" else D + 4


def work(case):
    if case["op"] == "logits":
        rows, vocab = case["requests"] * case["tokens"], case["vocab"]
        size = 2 if case["kind"] == "bf16" else 4
        n = rows * (2 * vocab * size + 4) + case["requests"] * 4 * (case["history"] + 2 * case["bias"])
        return {"bytes": n + (rows * 4 * (-(-vocab // 32)) if case["grammar"] else 0), "flops": 4 * rows * vocab}
    kv, cached = case["kv"], _row_bytes(case["kind"])
    if case["op"] == "read":
        rows = sum(_lengths(case)) * kv * 2
        return {"bytes": rows * cached + case["batch"] * case["ctx"] * kv * 2 * 2 * D, "flops": rows * D}
    new = case["batch"] * case["tokens"]
    if case["op"] == "append":
        return {"bytes": new * (case["heads"] * 4 * D + kv * 2 * (2 * D + cached)) + case["tokens"] * case["rot"] * 4,
                "flops": new * (case["heads"] + 2 * kv) * 4 * D}
    keys = sum(_lengths(case)) + new
    return {"bytes": new * case["heads"] * 4 * D + keys * kv * 2 * cached,
            "flops": 4 * D * case["heads"] * case["tokens"] * keys}


# ------------------------------------------------------------------ inputs
def _rope_table(n, rot):
    """cos | sin of every position, with the low frequencies stretched for long contexts."""
    i = torch.arange(0, rot, 2, dtype=torch.float64, device=DEV)
    inv = 500000.0 ** (-i / max(1, rot))
    turns = 8192 * inv / (2 * math.pi)
    keep = ((turns - 1.0) / 3.0).clamp(0, 1)
    inv = inv * keep + inv / 8.0 * (1 - keep)
    a = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.cat((a.cos(), a.sin()), 1).float()


def _trees(batch, tokens, seed):
    """Ancestor bits [batch, tokens, words] and depths [batch, tokens] of random trees; node 0 is the root."""
    r = random.Random(seed)
    words = -(-tokens // 64)
    bits, depth = [], []
    for _ in range(batch):
        anc, dep = [], []
        for i in range(tokens):
            p = i - 1 if i and r.random() < 0.4 else r.randrange(i) if i else -1
            anc.append((anc[p] if i else 0) | 1 << i)
            dep.append(dep[p] + 1 if i else 0)
        bits.append([[((a >> 64 * w & (1 << 64) - 1) ^ 1 << 63) - (1 << 63) for w in range(words)] for a in anc])
        depth.append(dep)
    return torch.tensor(bits, dtype=torch.int64, device=DEV), torch.tensor(depth, dtype=torch.int32, device=DEV)


def _quantised(x):
    scale = x.abs().amax(-1).clamp_min(1e-12) / E4M3_MAX
    return (x / scale[..., None]).to(F8), scale


def _pools(case, pages, gen):
    """K and V pages with rows in all of them (those behind a sequence's end are another's left-overs)."""
    out = {}
    for name in ("k", "v"):
        x = torch.randn(pages, case["kv"], PAGE, D, device=DEV, generator=gen)
        if case["kind"] == "bf16":
            out[name] = x.to(BF16)
        else:
            out[name], out[name + "_scale"] = _quantised(x)
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    if case["op"] == "logits":
        n, t, vocab, hist = (case[k] for k in ("requests", "tokens", "vocab", "history"))
        rows = n * t
        i32 = lambda lo, hi, *s: torch.randint(lo, hi, s, device=DEV, generator=gen, dtype=torch.int32)  # noqa: E731
        text = lambda *s: (vocab * torch.rand(*s, device=DEV, generator=gen) ** 3).int().clamp(max=vocab - 1)  # noqa: E731
        s = dict(logits=(4 * rnd(rows, vocab)).to(BF16 if case["kind"] == "bf16" else torch.float32),
                 requests=torch.arange(rows, dtype=torch.int32, device=DEV) // t, history=text(n, hist),
                 history_lens=i32(max(1, hist // 2), hist + 1, n), path=text(rows, t),
                 repetition=1 + 0.5 * torch.rand(n, device=DEV, generator=gen), frequency=0.5 * torch.rand(n, device=DEV, generator=gen),
                 presence=0.5 * torch.rand(n, device=DEV, generator=gen), bias_ids=None, bias=None, allowed=None)
        s["prompt_lens"] = (s["history_lens"] * torch.rand(n, device=DEV, generator=gen)).int()
        # a tree's rows have drafted between no and all of the tokens in front of them
        s["path"][torch.arange(t, device=DEV)[None] >= torch.arange(rows, device=DEV)[:, None] % t] = -1
        if case["bias"]:
            s["bias_ids"] = torch.rand(n, vocab, device=DEV, generator=gen).topk(case["bias"], dim=1).indices.int()
            s["bias"] = 5 * rnd(n, case["bias"])
        if case["grammar"]:      # about every fourth token is allowed
            words = (rows, -(-vocab // 32))
            s["allowed"] = i32(-2**31, 2**31 - 1, *words) & i32(-2**31, 2**31 - 1, *words)
        return dict(case=case, **s)
    lens = _lengths(case)
    random.Random(seed).shuffle(lens)
    tokens = case.get("tokens", 0)
    per = -(-(case["ctx"] + tokens) // PAGE)
    if case["op"] == "append":   # the new rows are the last ones
        lens = [n - min(n, tokens) for n in lens]
    pool = case["batch"] * per
    s = dict(case=case, lengths=torch.tensor(lens, dtype=torch.int32, device=DEV),
             pages=torch.randperm(pool, device=DEV, generator=gen).int().view(case["batch"], per))
    if case["op"] == "append":
        rows = rnd(case["batch"], tokens, case["heads"] + 2 * case["kv"], D).to(BF16)
        dims = (pool, case["kv"], PAGE, D)
        s.update({n: torch.zeros(dims, dtype=BF16 if case["kind"] == "bf16" else F8, device=DEV) for n in ("k", "v")})
        if case["kind"] == "e4m3":
            s.update({n: torch.zeros(dims[:3], device=DEV) for n in ("k_scale", "v_scale")})
        split = [case["heads"], case["kv"], case["kv"]]       # q, k and v as a fused projection leaves them
        s["new_q"], s["new_k"], s["new_v"] = rows.split(split, dim=2)
        s["table"] = _rope_table(case["ctx"] + tokens, case["rot"])
        s["norm"] = (1 + 0.1 * rnd(2, D)).to(BF16) if case["norm"] else None
        depth = _trees(case["batch"], tokens, seed)[1] if tokens <= 64 else torch.arange(tokens, dtype=torch.int32, device=DEV)
        s["positions"] = (s["lengths"][:, None] + depth).contiguous()
    else:
        s.update(_pools(case, pool, gen))
    if case["op"] == "attend":
        s["q"] = (1.5 * rnd(case["batch"], tokens, case["heads"], D)).to(BF16)
        s["mask"] = _trees(case["batch"], tokens, seed)[0]
    if own:
        from vdcores_b200 import ops
        s["cache"] = ops.KVCache(s["k"], s["v"], s.get("k_scale"), s.get("v_scale"))
    return s


# ------------------------------------------------------------------ the operators
def _pieces(kind):
    return 8 if kind == "bf16" else 16      # values of a 16-byte piece


def _swizzled(kind, row):
    """Place in a row of value d for rows `row` of a page: [..., 128]."""
    n, d = _pieces(kind), torch.arange(D, device=DEV)
    return ((d // n) ^ (row[..., None] & 7)) * n + d % n


def _rows(s, name):
    """The sequences' cache rows in fp32, [batch, rows, kv, 128], from the pages of the whole table."""
    kind = s["case"]["kind"]
    x = s[name][s["pages"].long()].float()                                      # [batch, pages, kv, 64, 128]
    x = x.gather(-1, _swizzled(kind, torch.arange(PAGE, device=DEV)).expand(x.shape))
    if kind == "e4m3":
        x = x * s[name + "_scale"][s["pages"].long()][..., None]
    return x.transpose(2, 3).flatten(1, 2)


def _plain_append(s):
    c = s["case"]
    rot, h = c["rot"], c["rot"] // 2
    cs = s["table"][s["positions"].long()][:, :, None]
    cos, sin = cs[..., :h], cs[..., h:]

    def turn(x, w):
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
        a, b = (x[..., :h], x[..., h:rot]) if c["layout"] == "half" else (x[..., :rot:2], x[..., 1:rot:2])
        pair = (a * cos - b * sin, b * cos + a * sin)
        y = torch.cat(pair, -1) if c["layout"] == "half" else torch.stack(pair, -1).flatten(-2)
        return torch.cat((y, x[..., rot:]), -1)

    norm = s["norm"] if s["norm"] is not None else (None, None)
    q = turn(s["new_q"].float(), norm[0]).to(BF16)
    at = s["lengths"].long()[:, None] + torch.arange(c["tokens"], device=DEV)
    page, row = s["pages"].long().gather(1, at // PAGE), at % PAGE
    place = _swizzled(c["kind"], row)[:, :, None]
    out = {"q": q}
    for name, x in (("k", turn(s["new_k"].float(), norm[1])), ("v", s["new_v"].float())):
        out[name] = s[name]
        if c["kind"] == "bf16":
            s[name][page, :, row] = x.to(BF16).gather(-1, place.expand(x.shape))
        else:
            code, scale = _quantised(x)
            s[name].view(torch.uint8)[page, :, row] = code.view(torch.uint8).gather(-1, place.expand(x.shape))
            s[name + "_scale"][page, :, row] = scale
            out[name + "_scale"] = s[name + "_scale"]
    return out


def _plain_read(s):
    n = s["case"]["ctx"]
    inside = (torch.arange(n, device=DEV) < s["lengths"][:, None])[..., None, None]
    return {name: torch.where(inside, _rows(s, name)[:, :n], 0.0).to(BF16) for name in ("k", "v")}


def _plain_attend(s):
    c = s["case"]
    t, g = c["tokens"], c["heads"] // c["kv"]
    k, v = _rows(s, "k"), _rows(s, "v")
    at = torch.arange(k.shape[1], device=DEV) - s["lengths"][:, None]           # place behind the context, [batch, rows]
    node = at.clamp(0, t - 1)
    bit = s["mask"].gather(2, (node // 64)[:, None].expand(-1, t, -1)) >> (node % 64)[:, None] & 1
    seen = (at < 0)[:, None] | ((at >= 0) & (at < t))[:, None] & bit.bool()     # [batch, t, rows]
    v = torch.where((at < t)[..., None, None], v, 0.0)
    q = s["q"].float().view(c["batch"], t, c["kv"], g, D).permute(0, 2, 1, 3, 4).flatten(2, 3)
    x = q @ k.permute(0, 2, 3, 1) * D ** -0.5
    x = torch.where(seen[:, None, :, None].expand(-1, -1, -1, g, -1).flatten(2, 3), x, -torch.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = x @ v.transpose(1, 2) / x.sum(-1, keepdim=True)
    return o.view(c["batch"], c["kv"], t, g, D).permute(0, 2, 1, 3, 4).reshape(s["q"].shape).to(BF16)


def _plain_logits(s):
    n, vocab = s["history"].shape[0], s["case"]["vocab"]
    req = s["requests"].long()
    at = torch.arange(s["history"].shape[1], device=DEV)
    table = lambda live: torch.zeros(n, vocab, dtype=torch.int32, device=DEV).scatter_add_(1, s["history"].long(), live.int())  # noqa: E731
    asked = table(at < s["prompt_lens"][:, None])
    count = table((at >= s["prompt_lens"][:, None]) & (at < s["history_lens"][:, None]))[req]
    count.scatter_add_(1, s["path"].clamp(min=0).long(), (s["path"] >= 0).int())
    x = s["logits"].float()
    rep = s["repetition"][req][:, None]
    x = torch.where((asked[req] > 0) | (count > 0), torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][req][:, None] * count
    x = x - s["presence"][req][:, None] * (count > 0)
    if s["bias"] is not None:
        x = x + torch.zeros(n, vocab, device=DEV).scatter_(1, s["bias_ids"].long(), s["bias"])[req]
    if s["allowed"] is not None:
        i = torch.arange(vocab, device=DEV)
        x = torch.where((s["allowed"][:, i // 32] >> (i % 32) & 1) > 0, x, -torch.inf)
    best = x.amax(1, keepdim=True)
    pick = torch.where(x == best, torch.arange(vocab, device=DEV), vocab).amin(1)
    return {"logits": x.to(s["logits"].dtype), "tokens": torch.where(best[:, 0] > -torch.inf, pick, -1).int()}


def run(s):
    c = s["case"]
    if not own:
        return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend, "logits": _plain_logits}[c["op"]](s)
    from vdcores_b200 import ops
    if c["op"] == "append":
        q = ops.rope_append(s["new_q"], s["new_k"], s["new_v"], s["cache"], s["pages"], s["lengths"], s["table"],
                            positions=s["positions"], layout=c["layout"], qk_norm=s["norm"])
        return {"q": q, **{n: s[n] for n in ("k", "v", "k_scale", "v_scale") if n in s}}
    if c["op"] == "read":
        k, v = ops.read_cache(s["cache"], s["pages"], s["lengths"], c["ctx"])
        return {"k": k, "v": v}
    if c["op"] == "attend":
        return ops.tree_attention(s["q"], s["cache"], s["pages"], s["lengths"], mask=s["mask"])
    logits, tokens = ops.adjust_logits(
        s["logits"], requests=s["requests"], history=s["history"], prompt_lens=s["prompt_lens"], history_lens=s["history_lens"],
        path=s["path"], repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"], bias_ids=s["bias_ids"],
        bias=s["bias"], allowed=s["allowed"])
    return {"logits": logits, "tokens": tokens}


# ------------------------------------------------------------------ the definitions in 64 bits
def _stored(s, name, b, n):
    """Rows 0 .. n - 1 of sequence b, [n, kv, 128] in 64 bits: every piece looked up where its row keeps it."""
    e = _pieces(s["case"]["kind"])
    i = torch.arange(n, device=DEV)
    page, row = s["pages"][b].long()[i // PAGE], i % PAGE
    x = s[name].double()[page, :, row].view(n, s["case"]["kv"], D // e, e)
    p = torch.arange(D // e, device=DEV)[None] ^ (row % 8)[:, None]
    x = torch.stack([x[i, :, p[:, j]] for j in range(D // e)], 2).flatten(2)
    return x * s[name + "_scale"].double()[page, :, row][..., None] if name + "_scale" in s else x


def _exact_append(s):
    c, r = s["case"], s["case"]["rot"]
    e = _pieces(c["kind"])
    out = {"q": None}
    ang = s["table"].double()[s["positions"].long()]
    z = torch.complex(ang[..., :r // 2], ang[..., r // 2:])[:, :, None]

    def turned(x, w):
        x = x.double()
        if s["norm"] is not None and w is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * w.double()
        y = x.clone()
        if c["layout"] == "half":
            p = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * z
            y[..., :r // 2], y[..., r // 2:r] = p.real, p.imag
        else:
            p = torch.complex(x[..., 0:r:2].contiguous(), x[..., 1:r:2].contiguous()) * z
            y[..., 0:r:2], y[..., 1:r:2] = p.real, p.imag
        return y

    w = s["norm"] if s["norm"] is not None else (None, None)
    out["q"] = turned(s["new_q"], w[0])
    for name, x in (("k", turned(s["new_k"], w[1])), ("v", s["new_v"].double())):
        pool = torch.zeros(s[name].shape, dtype=torch.float64, device=DEV)
        scales = torch.zeros(pool.shape[:3], dtype=torch.float64, device=DEV)
        for b in range(c["batch"]):
            i = int(s["lengths"][b]) + torch.arange(c["tokens"], device=DEV)
            page, row, y = s["pages"][b].long()[i // PAGE], i % PAGE, x[b]
            if c["kind"] == "e4m3":
                scale = y.abs().amax(-1).clamp_min(1e-12) / E4M3_MAX
                scales[page, :, row] = scale
                y = y / scale[..., None]
            for j in range(D // e):
                to = ((j ^ (row % 8)) * e)[:, None] + torch.arange(e, device=DEV)
                pool[page[:, None], :, row[:, None], to] = y[..., j * e:(j + 1) * e].transpose(1, 2)
        out[name] = pool
        if c["kind"] == "e4m3":
            out[name + "_scale"] = scales
    return out


def _exact_attend(s):
    c, t = s["case"], s["case"]["tokens"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    bits = s["mask"].cpu().tolist()
    for b in range(c["batch"]):
        n = int(s["lengths"][b])
        k, v = _stored(s, "k", b, n + t), _stored(s, "v", b, n + t)
        tree = torch.tensor([[bits[b][i][j // 64] >> j % 64 & 1 for j in range(t)] for i in range(t)], dtype=torch.bool, device=DEV)
        seen = torch.cat((torch.ones(t, n, dtype=torch.bool, device=DEV), tree), 1)
        for h in range(c["heads"]):
            kh = h // (c["heads"] // c["kv"])
            p = (s["q"][b, :, h].double() @ k[:, kh].t() / math.sqrt(D)).masked_fill(~seen, -math.inf).softmax(1)
            out[b, :, h] = p @ v[:, kh]
    return out


def _exact_logits(s):
    out = s["logits"].double()
    for r, n in enumerate(s["requests"].tolist()):
        x = out[r]
        asked, said = int(s["prompt_lens"][n]), int(s["history_lens"][n])
        words = torch.cat((s["history"][n, asked:said], s["path"][r][s["path"][r] >= 0])).long()
        count = torch.bincount(words, minlength=x.numel()).double()
        seen = count > 0
        seen[s["history"][n, :asked].long()] = True
        rep = s["repetition"][n].double()
        x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        x = x - s["frequency"][n].double() * count - s["presence"][n].double() * (count > 0).double()
        if s["bias"] is not None:
            x[s["bias_ids"][n].long()] += s["bias"][n].double()
        if s["allowed"] is not None:
            on = (s["allowed"][r][:, None].long() >> torch.arange(32, device=DEV) & 1).flatten()[:x.numel()]
            x[on == 0] = -math.inf
        out[r] = x
    return {"logits": out, "tokens": None}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "logits":
        return _exact_logits(s)
    out = {n: torch.zeros(case["batch"], case["ctx"], case["kv"], D, dtype=torch.float64, device=DEV) for n in ("k", "v")}
    for b, n in enumerate(s["lengths"].tolist()):
        for name in ("k", "v"):
            out[name][b, :n] = _stored(s, name, b, n)
    return out
