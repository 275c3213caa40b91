"""Operators for drafted tokens on the GPU, each against its formula in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F8, F64 = torch.bfloat16, torch.float8_e4m3fn, torch.float64
D, PAGE = 128, 64
U = 2.0 ** -8           # half a bf16 ulp, relative


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def swizzle(kind, rows):
    """Index [rows, 128]: value d of a page's row r is kept at [r, d]."""
    n, d = (8 if kind == "bf16" else 16), torch.arange(D)
    return ((d // n)[None] ^ (torch.as_tensor(rows) % 8)[:, None]) * n + (d % n)[None]


def rows_of(cache, pages_row, n, name):
    """Rows 0 .. n - 1 of a sequence, [n, heads, 128] in 64 bits (codes times scales)."""
    x, sc = getattr(cache, name), getattr(cache, name + "_scale")
    i = torch.arange(n)
    page, row = pages_row.cpu().long()[i // PAGE], i % PAGE
    to = lambda t: t.to(x.device)                                              # noqa: E731
    y = (x.view(F8) if cache.kind == "e4m3" else x)[to(page), :, to(row)].to(F64)
    y = y.gather(-1, to(swizzle(cache.kind, row))[:, None].expand(y.shape))
    return y * sc[to(page), :, to(row)].to(F64)[..., None] if sc is not None else y


def random_cache(dev, kind, n_pages, heads, seed):
    from vdcores_b200 import ops
    g = gen(dev, seed)
    x = [torch.randn(n_pages, heads, PAGE, D, device=dev, generator=g) for _ in range(2)]
    if kind == "bf16":
        return ops.KVCache(x[0].to(BF16), x[1].to(BF16))
    # scales that differ by a factor of a few hundred between rows
    s = [torch.exp(3 * torch.randn(n_pages, heads, PAGE, device=dev, generator=g).clamp(-1, 1)) * 0.01 for _ in range(2)]
    codes = [(t * 100).clamp(-448, 448).to(F8) for t in x]
    return ops.KVCache(codes[0], codes[1], s[0], s[1])


def page_table(dev, B, per, n_pages, seed):
    assert B * per <= n_pages
    return torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed))[:B * per].view(B, per).int().to(dev)


# ------------------------------------------------------------------ rope_append
def rope_reference(x, table, pos, layout, w, eps):
    """x [B, T, heads, 128] -> rotated, in 64 bits."""
    x = x.to(F64)
    if w is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.to(F64)
    rot = table.shape[1] if table is not None else 0
    if not rot:
        return x
    cs = table.to(F64)[pos.long()][:, :, None]
    c, s = cs[..., :rot // 2], cs[..., rot // 2:]
    i = torch.arange(rot // 2, device=x.device)
    a, b = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    y = x.clone()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("B,T,n_kv,group,layout,rot,norm,own_positions", [
    (1, 1, 8, 4, "half", 128, False, False),
    (1, 1, 1, 1, "interleaved", 128, False, True),
    (3, 5, 2, 4, "half", 32, True, True),
    (2, 130, 1, 8, "interleaved", 16, True, False),
    (2, 67, 3, 5, "half", 96, False, True),
    (4, 3, 4, 2, "interleaved", 0, True, False),
    (1, 2, 20, 16, "half", 64, True, True),
])
def test_rope_append(cuda_device, kind, B, T, n_kv, group, layout, rot, norm, own_positions):
    from vdcores_b200 import ops
    dev, g = cuda_device, gen(cuda_device, 1)
    per = 5
    cache = random_cache(dev, kind, B * per + 3, n_kv, 2)
    before = [t.clone() if t is not None else None for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    pages = page_table(dev, B, per, B * per + 3, 3)
    lengths = torch.randint(0, per * PAGE - T + 1, (B,), device=dev, generator=g, dtype=torch.int32)
    lengths[0] = 0
    counts = torch.randint(0, T + 1, (B,), device=dev, generator=g, dtype=torch.int32) if B > 1 else None
    # a fused projection's rows per KV head: [group queries | key | value], as the engines keep them
    fused = torch.randn(B, T, n_kv, group + 2, D, device=dev, generator=g).to(BF16)
    q, k, v = fused[..., :group, :], fused[..., group, :], fused[..., group + 1, :]
    table = ops.rope_table(per * PAGE + 10, rot, 1e4, device=dev) if rot else None
    pos = torch.randint(0, per * PAGE + 10, (B, T), device=dev, generator=g, dtype=torch.int32) if own_positions else None
    w = (1 + 0.3 * torch.randn(2, D, device=dev, generator=g)).to(BF16) if norm else None
    got = ops.rope_append(q, k, v, cache, pages, lengths, table, positions=pos, counts=counts, layout=layout, qk_norm=w, eps=1e-5)
    ops.check()

    at = lengths[:, None] + torch.arange(T, device=dev)
    turn = pos if pos is not None else at
    live = torch.arange(T, device=dev)[None] < (counts[:, None] if counts is not None else T)
    want_q = rope_reference(q.reshape(B, T, -1, D), table, turn, layout, w[0] if norm else None, 1e-5) * live[:, :, None, None]
    want = {"k": rope_reference(k, table, turn, layout, w[1] if norm else None, 1e-5), "v": v.to(F64)}
    # fp32 products and sums of values up to `top`: a few roundings of 2^-24 (the norm's sum of 128: more), then one to bf16
    fp32 = lambda x: 2.0 ** -18 * x.abs().amax(-1, keepdim=True)      # noqa: E731
    assert got.shape == q.shape
    err = (got.reshape(want_q.shape).to(F64) - want_q).abs()
    assert bool((err <= U * want_q.abs() + fp32(want_q)).all())
    written = torch.zeros(cache.k.shape[0], PAGE, dtype=torch.bool, device=dev)
    for b in range(B):
        for t in range(T):
            if not live[b, t]:
                continue
            page, row = int(pages[b, int(at[b, t]) // PAGE]), int(at[b, t]) % PAGE
            written[page, row] = True
    for name in ("k", "v"):
        for b in range(B):
            n = int(lengths[b]) + (int(counts[b]) if counts is not None else T)
            if n == int(lengths[b]):
                continue
            x, y = rows_of(cache, pages[b], n, name)[int(lengths[b]):], want[name][b][:n - int(lengths[b])]
            err = (x - y).abs()
            if kind == "bf16":
                assert bool((err <= U * y.abs() + fp32(y)).all())
            else:       # half an ulp of four significant bits, or half the smallest code, of a scale that is the maximum / 448
                scale = y.abs().amax(-1, keepdim=True) / 448
                assert bool((err <= 1.001 * (2.0 ** -4 * y.abs()).maximum(2.0 ** -10 * scale) + 2 * fp32(y)).all())
                # codes reach the top of the format, so nothing of it is given away
                assert bool(((x.abs().amax(-1) - y.abs().amax(-1)).abs() <= 2.0 ** -17 * y.abs().amax(-1)).all())
    # rows that are nobody's are as they were
    for t, old in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), before):
        if t is not None:
            same = (t.view(torch.uint8) if t.dtype == F8 else t) == (old.view(torch.uint8) if old.dtype == F8 else old)
            same = same.flatten(3).all(3) if same.dim() == 4 else same
            assert bool((same.all(1) | written).all())


def test_rope_append_in_place_and_through_an_engine_table(cuda_device):
    """out may be q; an engine's table (values rounded to bf16) is a table like any other."""
    from vdcores_b200 import ops
    dev, g = cuda_device, gen(cuda_device, 4)
    cache = random_cache(dev, "bf16", 4, 2, 5)
    pages = page_table(dev, 1, 2, 4, 6)
    table = ops.rope_table(128, device=dev).to(BF16).float()
    q, k, v = (torch.randn(1, 7, h, D, device=dev, generator=g).to(BF16) for h in (8, 2, 2))
    lengths = torch.tensor([61], dtype=torch.int32, device=dev)
    want = ops.rope_append(q, k, v, cache, pages, lengths, table)
    got = ops.rope_append(q, k, v, cache, pages, lengths, table, out=q)
    assert got is q and torch.equal(q, want)


def test_rope_append_rows_without_numbers(cuda_device):
    """Zero rows read back as zeros; a row with an infinity or NaN reads back without a number, and no other row does."""
    from vdcores_b200 import ops
    dev = cuda_device
    pages = torch.tensor([[0]], dtype=torch.int32, device=dev)
    lengths = torch.zeros(1, dtype=torch.int32, device=dev)
    k = torch.randn(1, 4, 1, D, device=dev, generator=gen(dev, 7)).to(BF16)
    v = k.flip(-1).contiguous()
    k[0, 1], v[0, 1] = 0, 0
    k[0, 2, 0, 5], v[0, 2, 0, 77] = math.inf, math.nan
    for kind in ("bf16", "e4m3"):
        cache = ops.KVCache.empty(1, 1, kind, dev)
        ops.rope_append(k, k, v, cache, pages, lengths)
        rk, rv = ops.read_cache(cache, pages, lengths + 4, 4)
        ops.check()
        for x, y in ((rk, k), (rv, v)):
            assert bool((x[0, 1] == 0).all())
            assert bool(x[0, [0, 1, 3]].isfinite().all())
            if kind == "bf16":
                assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))
            else:
                assert bool(x[0, 2].isnan().all())


# ------------------------------------------------------------------ read_cache
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("B,n_kv,n,lens,start", [
    (1, 8, 1, [1], None), (1, 1, 200, [0], None), (3, 2, 129, [128, 0, 129], None), (2, 3, 70, [300, 65], [5, 64]),
    (4, 4, 65, [64, 63, 1, 320], [0, 63, 7, 255])])
def test_read_cache(cuda_device, kind, B, n_kv, n, lens, start):
    from vdcores_b200 import ops
    dev, per = cuda_device, 5
    cache = random_cache(dev, kind, B * per + 1, n_kv, 11)
    pages = page_table(dev, B, per, B * per + 1, 12)
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    k, v = ops.read_cache(cache, pages, lengths, n, start=torch.tensor(start, dtype=torch.int32, device=dev) if start else None)
    ops.check()
    for name, got in (("k", k), ("v", v)):
        want = torch.zeros(B, n, n_kv, D, dtype=BF16, device=dev)
        for b in range(B):
            s = start[b] if start else 0
            m = max(0, min(n, lens[b] - s))
            if m:       # code * scale has at most 28 significant bits: fp32 rounds it once, bf16 once more, as here
                want[b, :m] = rows_of(cache, pages[b], s + m, name)[s:].float().to(BF16)
        assert torch.equal(got, want)


# ------------------------------------------------------------------ tree_attention
def attention_reference(q, cache, pages, lengths, seen, live, scale):
    """(outputs, sums of p |v|) in 64 bits; q [B, T, heads, 128], seen [B, T, T] bool, live [B]."""
    B, T, H, _ = q.shape
    out, mag = torch.zeros(q.shape, dtype=F64, device=q.device), torch.zeros(q.shape, dtype=F64, device=q.device)
    for b in range(B):
        n, m = int(lengths[b]), int(live[b])
        if n + m == 0 or m == 0:
            continue
        k, v = rows_of(cache, pages[b], n + m, "k"), rows_of(cache, pages[b], n + m, "v")
        ok = torch.cat((torch.ones(m, n, dtype=torch.bool, device=q.device), seen[b, :m, :m]), 1)
        for h in range(H):
            kh = h // (H // k.shape[1])
            s = (q[b, :m, h].to(F64) @ k[:, kh].t() * scale).masked_fill(~ok, -math.inf)
            p = torch.exp(s - s.amax(1, keepdim=True).clamp_min(-1e300)).masked_fill(~ok, 0)
            p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
            out[b, :m, h] = p @ v[:, kh]
            mag[b, :m, h] = p @ v[:, kh].abs()
    return out, mag


def assert_attention(got, want, mag):
    """One rounding of the weights to 8 significant bits or more, one of the result to bf16; scores off by a few 2^-24 of sums of
    128 products (2^-12 of a weight is more than that for scores below 100)."""
    err = (got.to(F64) - want).abs()
    bound = U * want.abs() + (U + 2.0 ** -12) * mag + 1e-30
    assert bool(got.isfinite().all()) and bool((err <= bound).all()), float((err / bound).max())


ATTENTION = [
    # B, T, n_kv, group, lengths, kind of mask
    (1, 1, 8, 4, [0], "chain"), (1, 1, 1, 1, [1], "chain"), (1, 1, 8, 4, [333], None), (2, 1, 2, 8, [64, 63], "chain"),
    (3, 7, 2, 4, [0, 57, 1000], "tree"), (2, 16, 8, 4, [120, 640], "tree"), (1, 33, 1, 1, [31], "tree"), (2, 64, 2, 4, [200, 0], "tree"),
    (1, 63, 4, 8, [2050], "tree"), (1, 130, 1, 3, [77], "tree"), (2, 100, 1, 8, [5, 129], None), (5, 3, 1, 5, [64, 128, 0, 61, 62], "random"),
    (1, 8, 2, 4, [20011], "chain"), (40, 2, 2, 4, None, "tree"), (1, 4, 1, 128, [300], "tree"), (1, 9, 3, 7, [448], "empty"),
    (3, 5, 2, 16, [0, 0, 0], "empty"),
]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_tree_attention(cuda_device, kind, case):
    from vdcores_b200 import ops
    dev, g = cuda_device, gen(cuda_device, case)
    B, T, n_kv, group, lens, how = ATTENTION[case]
    if lens is None:
        lens = [(i * 37) % 400 for i in range(B)]
    per = max(-(-(n + T) // PAGE) for n in lens) + 1
    cache = random_cache(dev, kind, B * per + 2, n_kv, 21)
    pages = page_table(dev, B, per, B * per + 2, 22)
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    q = torch.randn(B, T, n_kv * group, D, device=dev, generator=g).to(BF16)
    if how in (None, "chain"):
        seen = torch.ones(T, T, dtype=torch.bool, device=dev).tril().expand(B, T, T)
    elif how == "tree":
        parents = [[int(torch.randint(-1, i, (1,), device=dev, generator=g)) if i else -1 for i in range(T)] for _ in range(B)]
        seen = torch.zeros(B, T, T, dtype=torch.bool)
        for b in range(B):
            for i in range(T):
                seen[b, i] = seen[b, parents[b][i]] if parents[b][i] >= 0 else False
                seen[b, i, i] = True
        seen = seen.to(dev)
        assert torch.equal(ops.pack_mask(seen), ops.tree_mask(parents)[0])
    else:      # any token may see any other; in "empty" some rows see none
        seen = torch.rand(B, T, T, device=dev, generator=g) < 0.5
        if how == "empty":
            seen[:, ::2] = False
    mask = ops.pack_mask(seen) if how is not None else None
    # a batch's tail: every third sequence has drafted fewer tokens
    counts = torch.tensor([T - (i % 3) * T // 3 for i in range(B)], dtype=torch.int32, device=dev) if B > 2 else None
    live = counts if counts is not None else torch.full((B,), T)
    got = ops.tree_attention(q, cache, pages, lengths, mask=mask, counts=counts)
    ops.check()
    want, mag = attention_reference(q, cache, pages, lengths, seen, live, D ** -0.5)
    assert_attention(got, want, mag)
    again = ops.tree_attention(q, cache, pages, lengths, mask=mask, counts=counts)
    assert torch.equal(got, again)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_tree_attention_of_sharp_and_growing_scores(cuda_device, kind):
    """One key takes nearly all of the weight (first, last, or in the drafted tokens) while many small weights add up; and scores
    that grow from page to page, so that the running maximum moves all the time."""
    from vdcores_b200 import ops
    dev, g, n, T = cuda_device, gen(cuda_device, 31), 4000, 4
    per = -(-(n + T) // PAGE)
    pages = torch.arange(per, dtype=torch.int32, device=dev)[None]
    lengths = torch.tensor([n], dtype=torch.int32, device=dev)
    q = torch.randn(1, T, 4, D, device=dev, generator=g).to(BF16)
    u = q.double().mean((0, 1, 2))
    u = u / (q.double() @ u).abs().max() * D ** 0.5        # adds about 1 to the scores
    keys = 0.05 * torch.randn(1, n + T, 1, D, device=dev, generator=g).double()
    i = torch.arange(n + T, device=dev)
    for lift in ((i == 0) * 12.0, (i == n - 1) * 12.0, (i == n + 1) * 12.0, i * (60.0 / n), -i * (60.0 / n), ((i * 7919) % 997) / 30.0):
        cache = ops.KVCache.empty(per, 1, kind, dev)
        k = (keys + lift.double()[:, None, None] * u).to(BF16)
        v = torch.randn(1, n + T, 1, D, device=dev, generator=g).to(BF16)
        ops.rope_append(k, k, v, cache, pages, torch.zeros_like(lengths))
        got = ops.tree_attention(q, cache, pages, lengths)
        ops.check()
        seen = torch.ones(1, T, T, dtype=torch.bool, device=dev).tril()
        assert_attention(got, *attention_reference(q, cache, pages, lengths, seen, [T], D ** -0.5))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("T,group", [(5, 4), (20, 8), (1, 1)])
def test_tree_attention_ignores_what_is_masked(cuda_device, kind, T, group):
    """Left-overs behind a sequence's rows, drafted tokens that nobody sees, and pages that are not the sequence's may hold
    infinities and NaN; a seen token without numbers takes its number from those that see it, and from nobody else."""
    from vdcores_b200 import ops
    dev, g, n, per = cuda_device, gen(cuda_device, 41), 150, 4
    pages = torch.tensor([[5, 1, 4, 2]], dtype=torch.int32, device=dev)
    lengths = torch.tensor([n], dtype=torch.int32, device=dev)
    q = torch.randn(1, T, group, D, device=dev, generator=g).to(BF16)
    seen = torch.ones(1, T, T, dtype=torch.bool, device=dev).tril()
    poisoned = T // 2 if T > 1 else None
    if poisoned is not None:
        seen[:, :, poisoned] = False
    for bad in (math.nan, math.inf, -math.inf):
        cache = random_cache(dev, kind, 6, 1, 42)
        want = ops.tree_attention(q, cache, pages, lengths, mask=ops.pack_mask(seen))
        for at in [*range(n + T, per * PAGE), *([n + poisoned] if poisoned is not None else [])]:
            page, row = int(pages[0, at // PAGE]), at % PAGE
            for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
                if kind == "bf16":
                    x[page, :, row] = bad
                else:
                    x.view(torch.uint8)[page, :, row] = 0x7F      # NaN
                    s[page, :, row] = bad
        for x in (cache.k, cache.v):
            x.view(torch.uint8)[0] = 0xFF
            x.view(torch.uint8)[3] = 0xFF
        got = ops.tree_attention(q, cache, pages, lengths, mask=ops.pack_mask(seen))
        ops.check()
        assert torch.equal(got, want)
        if poisoned is not None:
            sees = seen.clone()
            sees[:, T - 1, poisoned] = True
            got = ops.tree_attention(q, cache, pages, lengths, mask=ops.pack_mask(sees))
            assert torch.equal(got[:, :T - 1], want[:, :T - 1])
            assert bool(got[:, T - 1].isnan().all())


def test_tree_attention_strides_scale_and_streams(cuda_device):
    """Queries and results as views with their own strides, one mask for all, shared pages, another scale, another stream."""
    from vdcores_b200 import ops
    dev, g, B, T, n_kv, group = cuda_device, gen(cuda_device, 51), 3, 6, 2, 4
    cache = random_cache(dev, "bf16", 9, n_kv, 52)
    pages = torch.tensor([[3, 4, 0], [3, 4, 1], [3, 8, 2]], dtype=torch.int32, device=dev)      # sequences share a prefix
    lengths = torch.tensor([130, 128, 100], dtype=torch.int32, device=dev)
    fused = torch.randn(B, T, n_kv, group + 2, D, device=dev, generator=g).to(BF16)
    q = fused[..., :group, :]
    parents = [-1, 0, 0, 1, 1, 4]
    mask, _ = ops.tree_mask(parents)
    wide = torch.full((B, T, 2, n_kv * group, D), 7.0, dtype=BF16, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.tree_attention(q, cache, pages, lengths, mask=mask, scale=0.3, out=wide[:, :, 1].unflatten(2, (n_kv, group)))
    torch.cuda.current_stream().wait_stream(side)
    ops.check()
    seen = torch.tensor([[bool(int(mask[i, 0]) >> j & 1) for j in range(T)] for i in range(T)], device=dev).expand(B, T, T)
    want, mag = attention_reference(q.reshape(B, T, -1, D), cache, pages, lengths, seen, [T] * B, 0.3)
    assert_attention(wide[:, :, 1], want, mag)
    assert got.shape == q.shape and bool((wide[:, :, 0] == 7).all())


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_pools_with_strides_and_offsets_beyond_32_bits(cuda_device, kind):
    """Layers side by side in one pool of more than 4 GiB; the pages used lie at both of its ends."""
    from vdcores_b200 import ops
    dev, g, n_kv = cuda_device, gen(cuda_device, 61), 2
    page_bytes = n_kv * PAGE * D * (2 if kind == "bf16" else 1)
    n_pages = (5 << 30) // (3 * page_bytes)
    pool = torch.empty(n_pages, 3, n_kv, PAGE, D, dtype=BF16 if kind == "bf16" else torch.uint8, device=dev)
    scale = torch.empty(n_pages, 3, n_kv, PAGE, device=dev) if kind == "e4m3" else None
    part = lambda t, i: t[:, i] if t is not None else None      # noqa: E731
    cache = ops.KVCache(part(pool, 0), part(pool, 2), part(scale, 0), part(scale, 2))
    pages = torch.tensor([[n_pages - 1, 0, n_pages - 2], [1, n_pages - 3, 2]], dtype=torch.int32, device=dev)
    n, T = 120, 9
    zero = torch.zeros(2, dtype=torch.int32, device=dev)
    k, v = (torch.randn(2, n + T, n_kv, D, device=dev, generator=g).to(BF16) for _ in range(2))
    q = torch.randn(2, n + T, n_kv * 4, D, device=dev, generator=g).to(BF16)
    ops.rope_append(q, k, v, cache, pages, zero)
    rk, _ = ops.read_cache(cache, pages, zero + n + T, n + T)
    out = ops.tree_attention(q[:, :T], cache, pages, zero + n)
    ops.check()
    assert float((rk.double() - k.double()).norm() / k.double().norm()) < (1e-12 if kind == "bf16" else 0.04)
    seen = torch.ones(2, T, T, dtype=torch.bool, device=dev).tril()
    assert_attention(out, *attention_reference(q[:, :T], cache, pages, zero + n, seen, [T, T], D ** -0.5))


def test_what_the_device_finds_wrong(cuda_device):
    """Pages, lengths and positions outside their ranges: the sequence is left out, the others are served, check() names it."""
    from vdcores_b200 import isa, ops, runtime
    dev, g = cuda_device, gen(cuda_device, 71)
    cache, other = random_cache(dev, "bf16", 4, 1, 72), random_cache(dev, "bf16", 4, 1, 72)     # one to read, one to write
    good = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=dev)
    lengths = torch.tensor([70, 20], dtype=torch.int32, device=dev)
    q, k, v = (torch.randn(2, 2, h, D, device=dev, generator=g).to(BF16) for h in (4, 1, 1))
    table = ops.rope_table(100, device=dev)
    ref = ops.tree_attention(q, cache, good, lengths)

    def wrong(word, fn):
        got = fn()
        with pytest.raises(runtime.VdcError, match=word) as e:
            ops.check()
        assert e.value.code == isa.ERR_RANGE
        ops.check()
        return got

    for value in (-1, 4, 2 ** 31 - 1):
        bad = good.clone()
        bad[0, 1] = value
        out = wrong("tree_attention: sequence 0: its page", lambda: ops.tree_attention(q, cache, bad, lengths))
        assert bool((out[0] == 0).all()) and torch.equal(out[1], ref[1])
        wrong("rope_append: sequence 0: its page", lambda: ops.rope_append(q, k, v, other, bad, lengths, table))
        rk, _ = wrong("read_cache: sequence 0: its page", lambda: ops.read_cache(cache, bad, lengths, 72))
        assert bool((rk[0, 64:] == 0).all())
    for value in (-1, 127, 2 ** 31 - 1):
        bad = lengths.clone()
        bad[0] = value
        out = wrong("tree_attention: sequence 0: its length", lambda: ops.tree_attention(q, cache, good, bad))
        assert bool((out[0] == 0).all()) and torch.equal(out[1], ref[1])
        wrong("rope_append: sequence 0: its length", lambda: ops.rope_append(q, k, v, other, good, bad, table if value < 0 else None))
    pos = torch.tensor([[3, 100], [0, 1]], dtype=torch.int32, device=dev)
    out = wrong("rope_append: sequence 0: its position", lambda: ops.rope_append(q, k, v, cache, good, lengths, table, positions=pos))
    assert bool((out[0, 1] == 0).all()) and bool((out[0, 0] != 0).any())


def test_refusals(cuda_device):
    from vdcores_b200 import ops
    dev = cuda_device
    bf = lambda *s: torch.zeros(*s, dtype=BF16, device=dev)      # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)      # noqa: E731
    cache = ops.KVCache.empty(4, 2, "bf16", dev)
    q, k, pages, lengths = bf(1, 3, 8, D), bf(1, 3, 2, D), i32(1, 2), i32(1)
    for fn in (
        lambda: ops.KVCache(bf(4, 2, 32, D), bf(4, 2, 32, D)), lambda: ops.KVCache(bf(4, 2, 64, D), bf(4, 1, 64, D)),
        lambda: ops.KVCache(bf(4, 2, 64, D).cpu(), bf(4, 2, 64, D).cpu()), lambda: ops.KVCache(bf(4, 2, 64, D), bf(4, 2, 64, D), bf(1), None),
        lambda: ops.KVCache(bf(4, 2, 64, D).view(torch.uint8)[..., :D], bf(4, 2, 64, D).view(torch.uint8)[..., :D]),
        lambda: ops.KVCache.empty(4, 2, "int8", dev),
        lambda: ops.tree_attention(q.float(), cache, pages, lengths), lambda: ops.tree_attention(bf(1, 3, 7, D), cache, pages, lengths),
        lambda: ops.tree_attention(bf(1, 3, 8, 64), cache, pages, lengths), lambda: ops.tree_attention(bf(2, 3, 8, D), cache, pages, lengths),
        lambda: ops.tree_attention(q, cache, pages.long(), lengths), lambda: ops.tree_attention(q, cache, pages, i32(2)),
        lambda: ops.tree_attention(q, cache, pages, lengths, mask=torch.zeros(1, 3, 2, dtype=torch.int64, device=dev)),
        lambda: ops.tree_attention(q, cache, pages, lengths, mask=torch.zeros(1, 3, 3, dtype=torch.bool, device=dev)),
        lambda: ops.tree_attention(q, cache, pages, lengths, out=q), lambda: ops.tree_attention(q, cache, pages.cpu(), lengths),
        lambda: ops.tree_attention(q, cache, pages, lengths, counts=i32(3)),
        lambda: ops.tree_attention(bf(1, 3, 8, 2 * D)[..., ::2], cache, pages, lengths),
        lambda: ops.rope_append(q, k, k, cache, pages, lengths, layout="both"), lambda: ops.rope_append(q, k, bf(1, 3, 1, D), cache, pages, lengths),
        lambda: ops.rope_append(q, k, k, cache, pages, lengths, positions=i32(1, 2)),
        lambda: ops.rope_append(q, k, k, cache, pages, lengths, table=bf(4, 128)),
        lambda: ops.rope_append(q, k, k, cache, pages, lengths, qk_norm=bf(D)), lambda: ops.read_cache(cache, pages, lengths, -1),
        lambda: ops.read_cache(cache, pages, lengths, 4, start=i32(2)),
        lambda: ops.adjust_logits(bf(2, 10).double()), lambda: ops.adjust_logits(bf(2, 10), history=i32(1, 4)),
        lambda: ops.adjust_logits(bf(2, 10), bias=torch.zeros(2, 1, device=dev)), lambda: ops.adjust_logits(bf(2, 10), allowed=i32(2, 2)),
        lambda: ops.adjust_logits(bf(2, 10), prompt_lens=i32(2)), lambda: ops.adjust_logits(bf(2, 10), out=torch.zeros(2, 10, dtype=torch.float16, device=dev)),
        lambda: ops.adjust_logits(bf(2, 10), repetition=bf(2)), lambda: ops.adjust_logits(bf(2, 20)[:, ::2]),
    ):
        with pytest.raises(ValueError):
            fn()
    from vdcores_b200 import runtime
    with pytest.raises(runtime.VdcError, match="multiple of 16"):
        ops.rope_append(q, k, k, cache, pages, lengths, table=torch.zeros(4, 24, device=dev))
    with pytest.raises(runtime.VdcError, match="misaligned"):
        ops.tree_attention(bf(1 * 3 * 8 * D + 1)[1:].view(1, 3, 8, D), cache, pages, lengths)
    # nothing to do
    assert ops.tree_attention(bf(0, 3, 8, D), cache, i32(0, 2), i32(0)).shape == (0, 3, 8, D)
    assert ops.tree_attention(bf(1, 0, 8, D), cache, pages, lengths).shape == (1, 0, 8, D)
    assert ops.rope_append(bf(1, 0, 8, D), bf(1, 0, 2, D), bf(1, 0, 2, D), cache, pages, lengths).shape == (1, 0, 8, D)
    assert ops.read_cache(cache, pages, lengths, 0)[0].shape == (1, 0, 2, D)
    assert ops.adjust_logits(bf(0, 10))[1].shape == (0,)
    ops.check()


# ------------------------------------------------------------------ adjust_logits
def logits_reference(x, req, history, prompt_lens, history_lens, path, rep, freq, pres, bias_ids, bias, allowed):
    """(adjusted logits in 64 bits, largest magnitude on the way)."""
    out, top = x.to(F64).cpu().clone(), x.to(F64).abs().cpu().clone()
    V = x.shape[1]
    for r in range(x.shape[0]):
        n = int(req[r])
        count, seen = [0] * V, [False] * V
        if rep is not None or freq is not None or pres is not None:
            h = history[n].tolist() if history is not None else []
            end = int(history_lens[n]) if history_lens is not None else len(h)
            first = int(prompt_lens[n]) if prompt_lens is not None else 0
            said = h[first:end] + (path[r].tolist() if path is not None else [])
            for t in h[:min(first, end)]:
                if 0 <= t < V:
                    seen[t] = True
            for t in said:
                if 0 <= t < V:
                    seen[t] = True
                    count[t] += 1
        for v in range(V):
            if seen[v]:
                if rep is not None:
                    out[r, v] = out[r, v] / float(rep[n]) if out[r, v] > 0 else out[r, v] * float(rep[n])
                if freq is not None:
                    out[r, v] -= float(freq[n]) * count[v]
                if pres is not None and count[v]:
                    out[r, v] -= float(pres[n])
                top[r, v] = max(float(top[r, v]), abs(float(out[r, v])), (float(freq[n]) if freq is not None else 0) * count[v])
        if bias_ids is not None:
            for t, w in zip(bias_ids[n].tolist(), bias[n].tolist()):
                if 0 <= t < V:
                    out[r, t] += w
                    top[r, t] += abs(w)
        if allowed is not None:
            words = allowed[r].tolist()
            for v in range(V):
                if not words[v // 32] >> (v % 32) & 1:
                    out[r, v] = -math.inf
    return out.to(x.device), top.to(x.device)


@pytest.mark.parametrize("dtype", [torch.float32, BF16, torch.float16])
@pytest.mark.parametrize("rows,n,V,L,p,m,grammar,strided", [
    (1, 1, 1, 3, 0, 0, False, False), (1, 1, 1001, 50, 0, 0, False, False), (7, 3, 513, 20, 4, 5, True, True), (3, 3, 40003, 300, 0, 3, True, False),
    (20, 5, 2048, 0, 6, 0, False, True), (2, 2, 131, 9, 1, 40, True, True), (300, 300, 77, 5, 0, 2, False, False)])
def test_adjust_logits(cuda_device, dtype, rows, n, V, L, p, m, grammar, strided):
    from vdcores_b200 import ops
    dev, g = cuda_device, gen(cuda_device, 81)
    i32 = lambda lo, hi, *s: torch.randint(lo, hi, s, device=dev, generator=g, dtype=torch.int32)      # noqa: E731
    x = 4 * torch.randn(rows, V + (3 if strided else 0), device=dev, generator=g)
    x = x.to(dtype)[:, 1:V + 1] if strided else x.to(dtype)
    req = i32(0, n, rows) if rows != n else torch.arange(rows, device=dev, dtype=torch.int32)
    kw = dict(history=i32(-1, V + 1, n, L) if L else None, prompt_lens=i32(0, L + 1, n) if L else None, history_lens=i32(0, L + 1, n) if L else None,
              path=i32(-1, min(V, 40), rows, p) if p else None)
    kw.update(repetition=1 + torch.rand(n, device=dev, generator=g), frequency=torch.rand(n, device=dev, generator=g),
              presence=torch.rand(n, device=dev, generator=g))
    if m:
        kw["bias_ids"], kw["bias"] = i32(-1, min(V, 30), n, m), 5 * torch.randn(n, m, device=dev, generator=g)
    if grammar:
        kw["allowed"] = i32(-2**31, 2**31 - 1, rows, -(-V // 32))
        kw["allowed"][0] = 0                                  # nothing is allowed
    if L:
        kw["prompt_lens"] = kw["prompt_lens"].minimum(kw["history_lens"])
    for out in (None, torch.full((rows, V + 5), 9.0, device=dev)[:, 2:V + 2]):
        got, tokens = ops.adjust_logits(x, requests=req if rows != n else None, out=out, **kw)
        ops.check()
        want, top = logits_reference(x, req, kw["history"], kw["prompt_lens"], kw["history_lens"], kw["path"], kw["repetition"],
                                     kw["frequency"], kw["presence"], kw.get("bias_ids"), kw.get("bias"), kw.get("allowed"))
        assert got.dtype == (dtype if out is None else torch.float32) and got.shape == x.shape
        assert torch.equal(got == -math.inf, want == -math.inf)
        fin = want > -math.inf
        # up to 5 + m fp32 roundings of values up to `top`, then one of the result
        bound = (5 + m) * 2.0 ** -24 * top + {torch.float32: 0.0, BF16: U, torch.float16: 2.0 ** -11}[got.dtype] * want.abs().nan_to_num(posinf=0, neginf=0) + 1e-7
        assert bool(((got.to(F64) - want).abs()[fin] <= bound[fin]).all())
        best = want.amax(1)
        for r in range(rows):
            if best[r] == -math.inf:
                assert int(tokens[r]) == -1
            else:
                assert float(want[r, int(tokens[r])]) >= float(best[r]) - 2 * float((5 + m) * 2.0 ** -24 * top[r].max()) - 1e-7
    # in place
    y = x.clone()
    got2, tokens2 = ops.adjust_logits(y, requests=req if rows != n else None, out=y, **kw)
    first, _ = ops.adjust_logits(x, requests=req if rows != n else None, **kw)
    assert got2 is y and torch.equal(y, first) and torch.equal(tokens, tokens2)


def test_adjust_logits_picks(cuda_device):
    """Ties go to the lowest id wherever they lie, NaN is never picked, infinities are; a row of NaN or of -inf has no pick; a vector
    is one row; whole numbers come through unchanged."""
    from vdcores_b200 import ops
    dev, V = cuda_device, 152000
    x = torch.zeros(6, V, dtype=BF16, device=dev)
    for r, at in enumerate(([5, 151999], [20000, 20001], [151999], [0, 77777])):
        x[r, at] = 3.0
    x[1, 100] = math.nan
    x[3, 9] = math.nan
    x[4] = math.nan
    x[5] = -math.inf
    out, tokens = ops.adjust_logits(x)
    assert tokens.tolist() == [5, 20000, 151999, 0, -1, -1]
    assert torch.equal(out.nan_to_num(5.0), x.nan_to_num(5.0))
    x[2, 3] = math.inf
    assert ops.adjust_logits(x)[1].tolist()[2] == 3
    out, tokens = ops.adjust_logits(x[0])
    assert out.shape == (V,) and tokens.tolist() == [5]
    assert torch.equal(out, x[0])
    # a drafted path counts like generated ids: 3 - 2 * 1 - 0.5 leaves the other maximum
    out, tokens = ops.adjust_logits(x[:1], path=torch.tensor([[5, 5]], dtype=torch.int32, device=dev), frequency=torch.ones(1, device=dev),
                                    presence=torch.full((1,), 0.5, device=dev))
    assert tokens.tolist() == [151999] and float(out[0, 5]) == 0.5
    # a long history of one id: the count does not wrap
    n = 70000
    out, _ = ops.adjust_logits(x[:1].float(), history=torch.full((1, n), 7, dtype=torch.int32, device=dev), frequency=torch.ones(1, device=dev))
    assert float(out[0, 7]) == -n
    ops.check()


def test_adjust_logits_reports_a_request_that_is_none(cuda_device):
    from vdcores_b200 import isa, ops, runtime
    dev = cuda_device
    x = torch.randn(3, 100, device=dev)
    for bad in (-1, 2):
        _, tokens = ops.adjust_logits(x, requests=torch.tensor([0, bad, 1], dtype=torch.int32, device=dev), repetition=torch.ones(2, device=dev))
        with pytest.raises(runtime.VdcError, match="row 1: its request") as e:
            ops.check()
        assert e.value.code == isa.ERR_RANGE and int(tokens[1]) == -1 and int(tokens[0]) == int(x[0].argmax())
