"""Operators for drafted tokens, what needs no GPU: rotation tables, tree masks, and the C ABI's refusals (arguments are looked at
before the device is)."""
import math

import pytest
import torch


def test_rope_table_follows_the_formulas():
    from vdcores_b200 import ops
    n, dim, theta = 50, 64, 1e4
    pos = torch.arange(n, dtype=torch.float64)[:, None]
    inv = torch.tensor([theta ** (-2 * i / dim) for i in range(dim // 2)], dtype=torch.float64)

    def table(freq, mag=1.0):
        return (mag * torch.cat(((pos * freq).cos(), (pos * freq).sin()), 1)).float()

    got = lambda s=None: ops.rope_table(n, dim, theta, s, device="cpu")      # noqa: E731
    # fp64 angles below 50 radians, one rounding to fp32: half an ulp of a value up to 1.2, and the angles' own 50 * 2^-52
    close = lambda a, b: torch.testing.assert_close(a, b, rtol=0, atol=2.0 ** -23)     # noqa: E731
    close(got(), table(inv))
    close(got({"type": "linear", "factor": 4.0}), table(inv / 4))
    close(got({"type": "ntk", "factor": 4.0}),
          table(torch.tensor([(theta * 4 ** (dim / (dim - 2))) ** (-2 * i / dim) for i in range(dim // 2)], dtype=torch.float64)))
    # llama3: every frequency by its turns in the original length
    lo, hi, f, orig = 1.0, 4.0, 8.0, 256
    out = []
    for v in inv.tolist():
        turns = orig * v / (2 * math.pi)
        keep = 0.0 if turns < lo else 1.0 if turns > hi else (turns - lo) / (hi - lo)
        out.append(v * keep + v / f * (1 - keep))
    assert out[-1] == inv[-1] / f and out[0] == inv[0]
    close(got({"type": "llama3", "factor": f, "low_freq_factor": lo, "high_freq_factor": hi, "original_max_position": orig}),
          table(torch.tensor(out, dtype=torch.float64)))
    # yarn: a ramp over the dimension, and a magnitude
    at = lambda turns: dim * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))    # noqa: E731
    a, b = max(math.floor(at(32)), 0), math.ceil(at(1))
    out = [v / f * r + v * (1 - r) for i, v in enumerate(inv.tolist()) for r in [min(max((i - a) / (b - a), 0), 1)]]
    close(got({"type": "yarn", "factor": f, "original_max_position": orig}), table(torch.tensor(out, dtype=torch.float64), 0.1 * math.log(f) + 1))


def test_rope_table_refusals():
    from vdcores_b200 import ops
    for bad in (dict(dim=24), dict(dim=144), dict(n_positions=0), dict(scaling={"type": "cubic"}), dict(scaling={"type": "linear", "factor": 0.5}),
                dict(scaling={"type": "linear", "factor": 2, "beta_fast": 1})):
        with pytest.raises(ValueError):
            ops.rope_table(**{"n_positions": 4, "device": "cpu", **bad})


@pytest.mark.parametrize("T", [1, 7, 64, 65, 130])
def test_tree_mask_names_every_ancestor(T):
    from vdcores_b200 import ops
    g = torch.Generator().manual_seed(T)
    parents = torch.stack([torch.tensor([int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for i in range(T)]) for _ in range(2)])
    mask, depth = ops.tree_mask(parents, device="cpu")
    assert mask.shape == (2, T, -(-T // 64)) and mask.dtype == torch.int64 and depth.dtype == torch.int32
    for b in range(2):
        for i in range(T):
            want, j = set(), i
            while j >= 0:
                want.add(j)
                j = int(parents[b, j])
            got = {j for j in range(T) if int(mask[b, i, j // 64]) >> (j % 64) & 1}
            assert got == want and int(depth[b, i]) == len(want) - 1
    one, d1 = ops.tree_mask(parents[0], device="cpu")
    assert torch.equal(one, mask[0]) and torch.equal(d1, depth[0])
    with pytest.raises(ValueError):
        ops.tree_mask([0])
    with pytest.raises(ValueError):
        ops.tree_mask([-1, 1])


def test_the_c_abi_refuses_without_a_gpu():
    import ctypes
    from vdcores_b200 import isa, runtime
    lib, base = runtime._lib, 1 << 20
    cache = runtime.Cache(base, base, base, base, 8192, 8192, 8192, 8192, 256, 256, 256, 256, 1, 2, 4, 0)

    def refused(fn, cls, good, word, **bad):
        a = cls()
        for k, v in {**good, **bad}.items():
            if k.startswith("cache_"):
                setattr(a.cache, k[6:], v)
            else:
                setattr(a, k, v)
        assert fn(ctypes.byref(a), 0, *([0] if cls is runtime.TreeAttention else [])) == isa.ERR_ARG
        assert word in runtime.last_error(), (bad, runtime.last_error())

    rope = dict(cache=cache, B=1, T=1, group=4, rot=128, table_rows=8, max_pages=4, q=base, k=base, v=base, out=base, pages=base,
                lengths=base, table=base)
    for word, bad in (("rotated part", dict(rot=24)), ("rotated part", dict(rot=144)), ("table", dict(table=0)), ("table", dict(table=base + 4)),
                      ("out of range", dict(T=0)), ("out of range", dict(B=-1)), ("out of range", dict(group=0)), ("rows", dict(q=0)),
                      ("rows", dict(v=base + 2)), ("strides", dict(k_t=4)), ("tables", dict(lengths=0)), ("tables", dict(counts=base + 1)),
                      ("kind", dict(cache_kind=2)), ("heads or pages", dict(cache_n_pages=0)), ("heads or pages", dict(max_pages=0)),
                      ("pages", dict(cache_k=base + 8)), ("pages", dict(cache_v_page=8)), ("scales", dict(cache_k_scale=0)),
                      ("scales", dict(cache_vs_head=4))):
        refused(lib.vdc_rope_append, runtime.RopeAppend, rope, word, **bad)
    read = dict(cache=cache, B=1, n=1, max_pages=4, pages=base, lengths=base, k_out=base, v_out=base)
    for word, bad in (("out of range", dict(n=0)), ("out of range", dict(B=0)), ("tables", dict(pages=0)), ("rows", dict(k_out=base + 4))):
        refused(lib.vdc_read_cache, runtime.ReadCache, read, word, **bad)
    tree = dict(cache=cache, B=1, T=65, group=4, max_pages=4, words=2, scale=1.0, q=base, out=base, pages=base, lengths=base, mask=base, work=base)
    for word, bad in (("out of range", dict(T=0)), ("out of range", dict(group=129)), ("fewer bits", dict(words=1)), ("rows", dict(out=0)),
                      ("strides", dict(o_t=4)), ("tables", dict(mask=base + 4)), ("tables", dict(pages=base + 2))):
        refused(lib.vdc_tree_attention, runtime.TreeAttention, tree, word, **bad)
    logit = dict(rows=2, vocab=10, n=2, logits=base, out=base, tokens=base)
    for word, bad in (("out of range", dict(rows=0)), ("out of range", dict(vocab=0)), ("out of range", dict(n_bias=1 << 20)),
                      ("types", dict(type=3)), ("types", dict(type=1, out_type=2)), ("logits", dict(out=base + 2)), ("logits", dict(logits=0)),
                      ("biases", dict(bias=base)), ("fewer requests", dict(n=1)), ("tables", dict(history=base + 2))):
        refused(lib.vdc_adjust_logits, runtime.AdjustLogits, logit, word, **bad)
    for fn in (lib.vdc_rope_append, lib.vdc_read_cache, lib.vdc_adjust_logits):
        assert fn(None, 0) == isa.ERR_ARG
