"""Decoding with drafted trees: every id must be a greedy choice of a plain fp64 model that is given the ids in front of it."""
import pytest
import torch

from oracle import decode_oracle as O
from tests.helpers import dense_weights, engine_config, perturb_norms, small_cfg

pytestmark = pytest.mark.gpu

PROMPTS = [[5, 9, 5, 9, 5, 9, 17], [3], list(range(40, 40 + 300)), [7, 7, 8] * 30]


def plain_logits(w, ids):
    """fp64 logits behind every id."""
    cfg = w.cfg
    f = lambda t: t.double()                                                               # noqa: E731
    norm = lambda x, g, eps: x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * f(g)  # noqa: E731
    T, d = len(ids), 128
    inv = cfg.theta ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    ang = torch.arange(T, dtype=torch.float64)[:, None] * inv
    cos, sin = (torch.cat((x, x), 1)[:, None] for x in (ang.cos(), ang.sin()))
    rot = lambda x: x * cos + torch.cat((-x[..., d // 2:], x[..., :d // 2]), -1) * sin     # noqa: E731
    h = f(w.embed)[torch.tensor(ids)]
    late = torch.ones(T, T, dtype=torch.bool).triu(1)
    for l in w.layers:
        x = norm(h, l.ln1, cfg.eps)
        q, k, v = ((x @ f(m.w).t()).view(T, -1, d) for m in (l.wq, l.wk, l.wv))
        if cfg.qk_norm:
            q, k = norm(q, l.q_norm, cfg.qk_norm_eps), norm(k, l.k_norm, cfg.qk_norm_eps)
        k, v = (y.repeat_interleave(cfg.n_heads // cfg.n_kv_heads, 1).transpose(0, 1) for y in (rot(k), v))
        s = (rot(q).transpose(0, 1) @ k.transpose(1, 2) / d ** 0.5).masked_fill(late, -torch.inf)
        h = h + (s.softmax(-1) @ v).transpose(0, 1).reshape(T, -1) @ f(l.wo.w).t()
        x = norm(h, l.ln2, cfg.eps)
        h = h + (torch.nn.functional.silu(x @ f(l.gate.w).t()) * (x @ f(l.up.w).t())) @ f(l.down.w).t()
    return norm(h, w.norm, cfg.eps) @ f(w.lm_head).t()


def assert_greedy(w, prompt, new, tol, repetition=1.0, frequency=0.0, presence=0.0):
    """Every new id's adjusted logit is within tol standard deviations of the largest."""
    ids = list(prompt) + list(new)
    logits = plain_logits(w, ids)
    for i in range(len(prompt), len(ids)):
        x = logits[i - 1].clone()
        sd = x.std()
        seen = torch.tensor(sorted(set(ids[:i])))
        times = torch.bincount(torch.tensor(ids[len(prompt):i], dtype=torch.long), minlength=len(x)).double()
        x[seen] = torch.where(x[seen] > 0, x[seen] / repetition, x[seen] * repetition)
        x = x - frequency * times - presence * (times > 0)
        assert x[ids[i]] >= x.max() - tol * sd, (i - len(prompt), ids[i], int(x.argmax()))


@pytest.fixture(scope="module", params=["llama", "qwen3"])
def model(request, cuda_device):
    from vdcores_b200.decode import DecodeEngine
    cfg = small_cfg(request.param)
    w = perturb_norms(O.ModelWeights.random(cfg, seed=3))
    eng = DecodeEngine(engine_config(cfg), max_seq=512)
    eng.load_weights(dense_weights(w))
    return w, eng


# bf16: some 30 roundings of 2^-9 a layer stack, under 2 % of a logit's deviation, five of which are allowed on top of each other; e4m3 rows:
# 2.5 % a value, so three times that
@pytest.mark.parametrize("kind, tol", [("bf16", 0.1), ("e4m3", 0.3)])
@pytest.mark.parametrize("branches, depth", [(0, 0), (2, 4), (3, 24)])
def test_ids_are_greedy(model, kind, tol, branches, depth):
    from vdcores_b200.drafted import DraftedDecoder
    w, eng = model
    dec = DraftedDecoder(eng, len(PROMPTS), 512, kind, branches, depth)
    dec.prefill(PROMPTS)
    new = dec.generate(24)
    assert all(len(x) == 24 for x in new) and dec.steps <= 24
    for prompt, ids in zip(PROMPTS, new):
        assert_greedy(w, prompt, ids, tol)


def test_penalties_count_drafted_ids(model):
    from vdcores_b200.drafted import DraftedDecoder
    w, eng = model
    how = dict(repetition=1.3, frequency=0.2, presence=0.3)
    dec = DraftedDecoder(eng, len(PROMPTS), 512, "bf16", 2, 4, **how)
    dec.prefill(PROMPTS)
    for prompt, ids in zip(PROMPTS, dec.generate(24)):
        assert_greedy(w, prompt, ids, 0.1, **how)


def test_the_second_branch_and_the_engine_go_on(model):
    """Drafts that are right in the second branch are accepted, their rows move, and the engine decodes behind them."""
    from vdcores_b200.drafted import DraftedDecoder
    w, eng = model
    plain = DraftedDecoder(eng, len(PROMPTS), 512, "bf16", 0, 0)
    plain.prefill(PROMPTS)
    known = [list(p) + x for p, x in zip(PROMPTS, plain.generate(40))]
    dec = DraftedDecoder(eng, len(PROMPTS), 512, "bf16", 2, 4)
    vocab, drafted = w.cfg.vocab, [0] * len(known)

    def draft(text):
        line = next((k for k in known if k[:len(text)] == text), None)
        if line:
            drafted[known.index(line)] += 1
        right = line[len(text):len(text) + 4] if line else []
        return [[(x + 1) % vocab for x in right], right] if len(right) == 4 else []
    dec.draft = draft
    dec.prefill(PROMPTS)
    new = dec.generate(24)
    for prompt, line, text, steps in zip(PROMPTS, known, dec.text, drafted):
        # five ids a step as long as the text is the known one (a near tie may fall the other way in a step of nine rows)
        same = next((i for i, (x, y) in enumerate(zip(line, text)) if x != y), min(len(line), len(text))) - len(prompt)
        assert steps <= same // 5 + 2
    for prompt, ids in zip(PROMPTS, new):
        assert_greedy(w, prompt, ids, 0.1)
    dec.hand_over(eng, 2)
    text = list(dec.text[2])
    assert_greedy(w, text, eng.generate(16), 0.1)


def test_refusals(model):
    from vdcores_b200.drafted import DraftedDecoder
    _, eng = model
    with pytest.raises(ValueError):
        DraftedDecoder(eng, 0, 64)
    with pytest.raises(ValueError):
        DraftedDecoder(eng, 1, 100000)
    dec = DraftedDecoder(eng, 1, 16, "bf16")
    with pytest.raises(ValueError):
        dec.prefill([[1], [2]])
    with pytest.raises(ValueError):
        dec.prefill([[]])
    dec.prefill([list(range(10))])
    with pytest.raises(RuntimeError):
        dec.generate(64)
