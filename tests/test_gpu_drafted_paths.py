"""What decides how the drafted-token operators go about their work: wide and narrow page tables, many and few rows, rows of one request in a
row or mixed, long texts, large vocabularies; and calls inside a CUDA graph."""
import math

import pytest
import torch

from tests.test_gpu_drafted import ATTENTION, assert_attention, attention_reference, gen, page_table, random_cache, rows_of

pytestmark = pytest.mark.gpu
BF16, F64, D, PAGE = torch.bfloat16, torch.float64, 128, 64
U = 2.0 ** -8


def tree_of(B, T, seed):
    g = torch.Generator().manual_seed(seed)
    seen = torch.zeros(B, T, T, dtype=torch.bool)
    for b in range(B):
        for i in range(T):
            p = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
            seen[b, i] = seen[b, p] if p >= 0 else False
            seen[b, i, i] = True
    return seen


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention_with_a_wide_page_table(cuda_device, kind, case):
    """A page table with room for many more rows than there are: units are divided among CTAs however short they are."""
    from vdcores_b200 import ops
    dev, (B, T, n_kv, group, lens, _) = cuda_device, ATTENTION[case]
    lens = [(i * 53) % 500 for i in range(B)] if lens is None else lens
    per = max(-(-(n + T) // PAGE) for n in lens)
    cache = random_cache(dev, kind, B * per, n_kv, 121)
    table = torch.full((B, per + 70), -1, dtype=torch.int32, device=dev)
    table[:, :per] = page_table(dev, B, per, B * per, 122)
    table[:, per:] = table[:, :1]
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    q = torch.randn(B, T, n_kv * group, D, device=dev, generator=gen(dev, case)).to(BF16)
    seen = tree_of(B, T, case).to(dev)
    counts = torch.tensor([T - (i % 3) * T // 3 for i in range(B)], dtype=torch.int32, device=dev)
    got = ops.tree_attention(q, cache, table, lengths, mask=ops.pack_mask(seen), counts=counts)
    ops.check()
    assert_attention(got, *attention_reference(q, cache, table, lengths, seen, counts, D ** -0.5))
    assert torch.equal(got, ops.tree_attention(q, cache, table, lengths, mask=ops.pack_mask(seen), counts=counts))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("B,T,n_kv,group,longest", [(41, 2, 8, 4, 2500), (41, 2, 8, 4, 700), (170, 1, 2, 7, 130), (25, 40, 8, 2, 300)])
def test_attention_of_many_units(cuda_device, kind, B, T, n_kv, group, longest):
    """More units than SMs, of lengths from nothing to many pages."""
    from vdcores_b200 import ops
    dev = cuda_device
    lens = [(i * 7919) % longest for i in range(B - 1)] + [longest]
    per = -(-(longest + T) // PAGE)
    cache = random_cache(dev, kind, B * per, n_kv, 131)
    pages = page_table(dev, B, per, B * per, 132)
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    q = torch.randn(B, T, n_kv * group, D, device=dev, generator=gen(dev, B)).to(BF16)
    seen = torch.ones(T, T, dtype=torch.bool, device=dev).tril().expand(B, T, T)
    counts = torch.tensor([(i * 5) % (T + 1) for i in range(B)], dtype=torch.int32, device=dev)
    got = ops.tree_attention(q, cache, pages, lengths, counts=counts)
    ops.check()
    assert_attention(got, *attention_reference(q, cache, pages, lengths, seen, counts, D ** -0.5))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("B,T", [(1, 1), (40, 16), (3, 900)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_append_of_few_and_many_tokens(cuda_device, kind, B, T, layout):
    """One and the same row whatever the number of tokens it comes with."""
    from vdcores_b200 import ops
    dev, n_kv, group = cuda_device, 3, 5
    g = gen(dev, 141)
    q, k, v = (torch.randn(B, T, h, D, device=dev, generator=g).to(BF16) for h in (n_kv * group, n_kv, n_kv))
    per = -(-(T + 30) // PAGE)
    table = ops.rope_table(T + 40, 96)
    lengths = torch.tensor([i % 30 for i in range(B)], dtype=torch.int32, device=dev)
    pages = page_table(dev, B, per, B * per, 142)
    cache = ops.KVCache.empty(B * per, n_kv, kind, dev)
    out = ops.rope_append(q, k, v, cache, pages, lengths, table, layout=layout)
    for b, t in {(0, 0), (B - 1, T - 1), (B // 2, T // 2)}:
        one = ops.KVCache.empty(per, n_kv, kind, dev)
        row = pages[:1] * 0 + torch.arange(per, dtype=torch.int32, device=dev)
        at = lengths[b:b + 1] + t
        o = ops.rope_append(q[b:b + 1, t:t + 1], k[b:b + 1, t:t + 1], v[b:b + 1, t:t + 1], one, row, at, table, layout=layout)
        assert torch.equal(o[0, 0], out[b, t])
        n = int(at) + 1
        for name in "kv":
            assert torch.equal(rows_of(one, row[0], n, name)[-1], rows_of(cache, pages[b], n, name)[-1])
    ops.check()


def logits_in_64_bits(x, req, history, prompt_lens, history_lens, path, rep, freq, pres, bias_ids, bias, allowed):
    n, V, dev = len(rep), x.shape[1], x.device
    inside = lambda t: (t >= 0) & (t < V)                                                     # noqa: E731
    table = lambda ids, live: torch.zeros(len(ids), V, device=dev).scatter_add_(             # noqa: E731
        1, ids.long().clamp(0, V - 1), (inside(ids) & live).float())
    at = torch.arange(history.shape[1], device=dev)
    said = table(history, (at >= prompt_lens[:, None]) & (at < history_lens[:, None]))[req.long()] + table(path, path >= 0)
    seen = (said > 0) | (table(history, at < prompt_lens[:, None])[req.long()] > 0)
    r, f, p = (t.to(F64)[req.long()][:, None] for t in (rep, freq, pres))
    y = x.to(F64)
    y = torch.where(seen, torch.where(y > 0, y / r, y * r), y) - f * said - p * (said > 0)
    add = torch.zeros(n, V, dtype=F64, device=dev).scatter_add_(1, bias_ids.long().clamp(0, V - 1), bias.to(F64) * inside(bias_ids))
    y = y + add[req.long()]
    may = (allowed.long()[:, :, None] >> torch.arange(32, device=dev) & 1).flatten(1)[:, :V].bool()
    return y.masked_fill(~may, -math.inf)


# rows, requests, vocabulary, text, path, how the rows' requests come, elements between rows beyond the vocabulary
@pytest.mark.parametrize("rows,n,V,L,p,how,pad", [
    (640, 80, 4099, 50, 6, "runs", 0), (640, 80, 4099, 50, 6, "runs", 5), (700, 9, 1030, 200, 3, "mixed", 2), (640, 64, 513, 20, 70, "runs", 0),
    (3, 2, 40001, 13000, 4, "mixed", 3), (2, 2, 300007, 13000, 2, "runs", 0), (330, 7, 300007, 30, 2, "runs", 1), (1, 1, 9, 9000, 1, "runs", 0),
    (2, 1, 16, 4, 64, "runs", 0)])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_adjust_logits_paths(cuda_device, rows, n, V, L, p, how, pad, dtype):
    from vdcores_b200 import ops
    dev, g = cuda_device, gen(cuda_device, rows + V)
    i32 = lambda lo, hi, *s: torch.randint(lo, hi, s, device=dev, generator=g, dtype=torch.int32)      # noqa: E731
    x = (4 * torch.randn(rows, V + pad, device=dev, generator=g)).to(dtype)[:, :V]
    req = torch.arange(rows, device=dev, dtype=torch.int32) * n // rows if how == "runs" else i32(0, n, rows)
    lens = i32(0, L + 1, n)
    kw = dict(history=i32(-2, V + 2, n, L), history_lens=lens, prompt_lens=(lens * torch.rand(n, device=dev, generator=g)).int(),
              path=i32(-1, V + 1, rows, p), repetition=1 + torch.rand(n, device=dev, generator=g), frequency=torch.rand(n, device=dev, generator=g),
              presence=torch.rand(n, device=dev, generator=g), bias_ids=i32(-1, V + 1, n, 5), bias=torch.randn(n, 5, device=dev, generator=g),
              allowed=i32(-2**31, 2**31 - 1, rows, -(-V // 32)))
    kw["path"][::3] = kw["history"][req.long()[::3], :1]            # some ids again and again
    kw["bias_ids"][:, 4] = kw["bias_ids"][:, 0]                     # two biases of one id
    got, tokens = ops.adjust_logits(x, requests=req, **kw)
    ops.check()
    want = logits_in_64_bits(x, req, *(kw[k] for k in ("history", "prompt_lens", "history_lens", "path", "repetition", "frequency", "presence",
                                                       "bias_ids", "bias", "allowed")))
    assert torch.equal(got == -math.inf, want == -math.inf)
    fin = want > -math.inf
    # ten fp32 roundings of values on the way that stay below 2^15 (a thousand of one id at most, in these texts), one of the result
    bound = 10 * 2.0 ** -24 * 2.0 ** 15 * (kw["history"].shape[1] > 1000) + 10 * 2.0 ** -24 * 256 + (U if dtype == BF16 else 0) * want.abs()
    assert bool(((got.to(F64) - want).abs()[fin] <= bound[fin]).all())
    best = want.amax(1)
    chosen = want.gather(1, tokens.long().clamp(min=0)[:, None])[:, 0]
    assert torch.equal(tokens < 0, best == -math.inf)
    ok = tokens >= 0
    assert bool((chosen[ok] >= best[ok] - 2.0 ** -6).all())
    alone, token = ops.adjust_logits(x[-1:], requests=req[-1:], **{k: t[-1:] if k in ("path", "allowed") else t for k, t in kw.items()})
    assert torch.equal(alone[0], got[-1]) and int(token) == int(tokens[-1])


def test_calls_in_a_graph(cuda_device):
    """The four operators captured once and replayed on other contents: the same as outside."""
    from vdcores_b200 import ops
    dev, B, T, n_kv, group, V = cuda_device, 3, 8, 2, 4, 5000
    for per in (4, 90):                         # units whole and divided
        cache = ops.KVCache.empty(B * per, n_kv, "e4m3", dev)
        pages = page_table(dev, B, per, B * per, 151)
        table = ops.rope_table(per * PAGE)
        lengths = torch.zeros(B, dtype=torch.int32, device=dev)
        mask = ops.pack_mask(tree_of(B, T, 5).to(dev))
        q, k, v = (torch.zeros(B, T, h, D, dtype=BF16, device=dev) for h in (n_kv * group, n_kv, n_kv))
        logits = torch.zeros(B * T, V, dtype=BF16, device=dev)
        history = torch.zeros(B, 30, dtype=torch.int32, device=dev)
        req = torch.arange(B * T, dtype=torch.int32, device=dev) // T
        rep = torch.full((B,), 1.5, device=dev)

        def run():
            turned = ops.rope_append(q, k, v, cache, pages, lengths, table)
            o = ops.tree_attention(turned, cache, pages, lengths, mask=mask)
            y, tokens = ops.adjust_logits(logits, requests=req, history=history, repetition=rep)
            return (turned, o, y, tokens) + ops.read_cache(cache, pages, lengths + T, 100)

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = run()
        for seed in range(3):
            g = gen(dev, 160 + seed)
            for t in (q, k, v, logits):
                t.copy_(torch.randn(t.shape, device=dev, generator=g))
            history.copy_(torch.randint(0, V, history.shape, device=dev, generator=g))
            lengths.copy_(torch.randint(0, (min(per, 40) - 1) * PAGE, (B,), device=dev, generator=g))
            graph.replay()
            got = [t.clone() for t in held]
            want = run()
            ops.check()
            assert all(torch.equal(x, y) for x, y in zip(got, want))
