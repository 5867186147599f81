"""A model with a paged cache (elb_model_set_pages) against the same model with the contiguous one: prompts, turns and batched steps of
several sequences, forks and beam searches (elb_model_reorder, elb_model_eval_batch_beam), pages running out, refusals."""
import numpy as np
import pytest

import exactinfer_b200 as e
import oracle_lib as ol
from exactinfer_b200 import synth

pytestmark = pytest.mark.gpu
REL_TOL = 2e-4  # the bar of the batch tests: the pair cache holds 22 bits, the attention's operands as well
# fp16 pages, against 64 bits with the same rounding of keys and values: the two sides' values differ by some 1e-5 before it, so that
# one in fifty ends a step of 2^-11 away; a score of 128 products then differs by about sqrt(128 / 50) * 2^-11 / sqrt(128) * |q k|,
# 7e-5 times the largest products (about 10), and two layers pass it on a few times
REL_F16 = 8e-3


@pytest.fixture(scope="module", autouse=True)
def device():
    ok, why = e.cuda_available()
    assert ok, f"CUDA path unavailable: {why}"


def spec_of(layout, **kw):
    return synth.Spec(**(dict(name="paged", n_layer=2, n_embd=512, n_ff=1024, n_head=8, n_head_kv=2, n_vocab=1200, layout=layout, head_sigma=2e-5) | kw))


@pytest.fixture(scope="module", params=("q4_k_m", "f16"))
def models(request):
    spec = spec_of(request.param)
    tens = list(synth.generate(spec, 17))
    make = lambda **kw: e.Backend(spec, tens, 96, max_batch=32, n_seq=6, **kw)
    return spec, make, make()


def rel(a, b):
    return float(np.abs(a.astype(np.float64) - b).max() / np.abs(b).max())


def prompt(model, s, toks, pos0=0):
    if len(toks) > 32:  # (max_batch)
        prompt(model, s, toks[:-8], pos0)
        return prompt(model, s, toks[-8:], pos0 + len(toks) - 8)
    want = np.zeros(len(toks), np.uint8)
    want[-1] = 1
    return model.eval_batch(toks, np.full(len(toks), s), np.arange(pos0, pos0 + len(toks)), want)[0]


@pytest.mark.parametrize("pages", [(16, 24, e.KV_PAIR), (32, 18, e.KV_PAIR)])
def test_paged_model_equals_contiguous_model(models, pages):
    spec, make, flat = models
    tol = REL_TOL
    paged = make(pages=pages)
    rng = np.random.default_rng(5)
    pos = [0] * 4
    for s, n in enumerate((23, 1, 16, 30)):
        toks = rng.integers(0, spec.n_vocab, n)
        assert rel(prompt(paged, s, toks), prompt(flat, s, toks)) <= tol
        pos[s] = n
    for step in range(6):  # steps of all sequences in changing order, with a turn of several rows among them
        rows = [(s, 1 if (s + step) % 4 else 5) for s in rng.permutation(4)]
        seq = [s for s, n in rows for _ in range(n)]
        ps = [pos[s] + i for s, n in rows for i in range(n)]
        if step % 2:  # rows of different sequences between one another
            mix = sorted(range(len(seq)), key=lambda i: (ps[i] - pos[seq[i]], i))
            seq, ps = [seq[i] for i in mix], [ps[i] for i in mix]
        toks = rng.integers(0, spec.n_vocab, len(seq))
        want = np.array([p == pos[s] + dict(rows)[s] - 1 for s, p in zip(seq, ps)], np.uint8)
        a, b = paged.eval_batch(toks, seq, ps, want), flat.eval_batch(toks, seq, ps, want)
        assert rel(a, b) <= tol
        ta, tb = paged.eval_batch_top(toks, seq, ps, 3, want), flat.eval_batch_top(toks, seq, ps, 3, want)
        assert rel(ta[1], tb[1]) <= tol and np.abs(ta[2] - tb[2]).max() <= tol * np.abs(tb[1]).max()
        assert rel(paged.hidden(), flat.hidden()) <= tol
        for s, n in rows:
            pos[s] += n
    held = sum(-(-p // pages[0]) for p in pos)
    assert paged.free_pages() == pages[1] - held
    paged.drop(3)
    assert paged.free_pages() == pages[1] - held + -(-pos[3] // pages[0])


def rounded_logits(spec, tens, toks):
    """The forward pass in 64 bits with keys (behind the rotation) and values rounded to fp16, last token's logits."""
    T = {(r, l): (t, rows, n, w) for r, l, t, rows, n, w in tens}

    def W(role, l):
        t, rows, n, w = T[(role, l)]
        return np.ascontiguousarray(w).view(np.float32).reshape(-1).astype(np.float64) if t == synth.F32 else ol.dequant_rows(t, rows, n, w).astype(np.float64)

    rms = lambda v, w: v / np.sqrt((v * v).mean(-1, keepdims=True) + spec.eps) * w
    half = lambda a: a.astype(np.float16).astype(np.float64)
    emb = W("token_embd", -1)
    x, n, H, K, D = emb[toks], len(toks), spec.n_head, spec.n_head_kv, spec.head_dim
    th = np.arange(n)[:, None] * spec.rope_base ** (-2.0 * np.arange(D // 2) / D)[None]
    c, s = np.cos(th)[:, None], np.sin(th)[:, None]
    turn = lambda a: np.concatenate([a[..., :D // 2] * c - a[..., D // 2:] * s, a[..., :D // 2] * s + a[..., D // 2:] * c], -1)
    for l in range(spec.n_layer):
        h = rms(x, W("attn_norm", l))
        q, k, v = (np.reshape(h @ W(r, l).T, (n, m, D)) for r, m in (("attn_q", H), ("attn_k", K), ("attn_v", K)))
        q, k, v = turn(rms(q, W("attn_q_norm", l))), half(turn(rms(k, W("attn_k_norm", l)))), half(v)
        sc = np.einsum("ihd,jhd->hij", q, np.repeat(k, H // K, 1)) / np.sqrt(D)
        sc = np.where(np.tril(np.ones((n, n), bool)), sc, -np.inf)
        p = np.exp(sc - sc.max(-1, keepdims=True))
        out = np.einsum("hij,jhd->ihd", p / p.sum(-1, keepdims=True), np.repeat(v, H // K, 1))
        x = x + out.reshape(n, H * D) @ W("attn_output", l).T
        h = rms(x, W("ffn_norm", l))
        g, u = h @ W("ffn_gate", l).T, h @ W("ffn_up", l).T
        x = x + (g / (1 + np.exp(-g)) * u) @ W("ffn_down", l).T
    return rms(x[-1], W("output_norm", -1)) @ emb.T


def test_fp16_pages(models):
    spec, make, _ = models
    tens = list(synth.generate(spec, 17))
    paged = make(pages=(16, 24, e.KV_F16))
    rng = np.random.default_rng(12)
    hist = [rng.integers(0, spec.n_vocab, n) for n in (21, 30)]
    for s, toks in enumerate(hist):
        assert rel(prompt(paged, s, toks), rounded_logits(spec, tens, toks)) <= REL_F16
    for step in range(3):
        nxt = rng.integers(0, spec.n_vocab, 2)
        out = paged.eval_batch(nxt, [1, 0], [len(hist[1]), len(hist[0])])
        hist = [np.append(hist[0], nxt[1]), np.append(hist[1], nxt[0])]
        for r, s in enumerate((1, 0)):
            assert rel(out[r], rounded_logits(spec, tens, hist[s])) <= REL_F16


def test_single_sequence_calls(models):
    spec, make, flat = models
    paged = make(pages=(16, 12, e.KV_PAIR))
    rng = np.random.default_rng(6)
    toks = rng.integers(0, spec.n_vocab, 75)  # three chunks of 32
    assert rel(paged.eval(toks, 0), flat.eval(toks, 0)) <= REL_TOL
    nxt = rng.integers(0, spec.n_vocab, 4)
    for i in range(3):
        assert rel(paged.eval(nxt[i:i + 1], 75 + i), flat.eval(nxt[i:i + 1], 75 + i)) <= REL_TOL
    allowed = rng.random(spec.n_vocab) < 0.2
    a, b = paged.eval_top(nxt[3:], 78, 5, allowed), flat.eval_top(nxt[3:], 78, 5, allowed)
    assert (a[0] == b[0]).all() and abs(a[2] - b[2]) <= REL_TOL * np.abs(b[1]).max()
    assert paged.eval_steps(nxt, 79) > 0
    # back into the middle: what follows is cut off
    assert rel(paged.eval(nxt[:2], 20), flat.eval(nxt[:2], 20)) <= REL_TOL
    assert paged.free_pages() == 12 - 2
    with pytest.raises(IndexError):
        paged.eval(nxt[:1], 23)  # a hole
    assert rel(paged.eval(nxt[:1], 22), flat.eval(nxt[:1], 22)) <= REL_TOL


def test_forks_share_pages_and_do_not_disturb_each_other(models):
    spec, make, flat = models
    paged = make(pages=(16, 14, e.KV_PAIR))
    rng = np.random.default_rng(7)
    toks = rng.integers(0, spec.n_vocab, 37)  # two full pages and 5 positions
    prompt(paged, 2, toks)
    assert paged.free_pages() == 11
    paged.reorder([0, 1, 3], [2, 2, 2])  # one of the four keeps the last page, three copies
    assert paged.free_pages() == 8
    for s in range(4):
        prompt(flat, s, toks)
    for step in range(14):  # over the end of the page
        nxt = rng.integers(0, spec.n_vocab, 4)
        a, b = paged.eval_batch(nxt, range(4), [37 + step] * 4), flat.eval_batch(nxt, range(4), [37 + step] * 4)
        assert rel(a, b) <= REL_TOL
    assert paged.free_pages() == 14 - (2 + 4 + 4)
    # into a shared page: the writer gets one of its own, the others keep theirs
    nxt = rng.integers(0, spec.n_vocab, 3)
    assert rel(prompt(paged, 1, nxt, 20), prompt(flat, 1, nxt, 20)) <= REL_TOL
    nxt = rng.integers(0, spec.n_vocab, 3)
    seq = [0, 2, 3]
    assert rel(paged.eval_batch(nxt, seq, [51] * 3), flat.eval_batch(nxt, seq, [51] * 3)) <= REL_TOL
    for s in range(4):
        paged.drop(s)
    assert paged.free_pages() == 14


def test_reorder_swaps_and_empty_parents(models):
    spec, make, flat = models
    paged = make(pages=(16, 20, e.KV_PAIR))
    rng = np.random.default_rng(8)
    toks = [rng.integers(0, spec.n_vocab, n) for n in (20, 33)]
    for s in range(2):
        prompt(paged, s, toks[s])
        prompt(flat, 1 - s, toks[s])
    paged.reorder([0, 1, 5], [1, 0, 4])  # 4 holds nothing
    nxt = rng.integers(0, spec.n_vocab, 2)
    assert rel(paged.eval_batch(nxt, [0, 1], [33, 20]), flat.eval_batch(nxt, [0, 1], [33, 20])) <= REL_TOL
    assert paged.free_pages() == 20 - 3 - 2
    paged.reorder([], [])
    paged.reorder([0, 1], [4, 4])
    assert paged.free_pages() == 20


def test_beam_search_finds_what_a_plain_search_finds(models):
    """Two prompts, three beams each, end to end: the device's picks over its own logits, and every beam's logits are those of its
    tokens evaluated from the start."""
    spec, make, flat = models
    beams, steps = 3, 6
    paged = make(pages=(16, 40, e.KV_PAIR))
    rng = np.random.default_rng(9)
    toks = [rng.integers(0, spec.n_vocab, n) for n in (14, 9)]
    # first step: the last rows of the two prompts, one live beam each
    seq = np.concatenate([np.full(len(t), g * beams) for g, t in enumerate(toks)])
    pos = np.concatenate([np.arange(len(t)) for t in toks])
    want = np.zeros(seq.size, np.uint8)
    want[[13, 22]] = 1
    parent, token, score = paged.eval_batch_beam(np.concatenate(toks), seq, pos, [0.0, 0.0], 1, beams, want)
    paged.reorder(range(6), [g * beams for g in range(2) for _ in range(beams)])
    hist = [[int(token[g, b])] for g in range(2) for b in range(beams)]
    scores = score.reshape(-1)
    for step in range(steps):
        length = [len(toks[r // beams]) + step for r in range(6)]
        last = [h[-1] for h in hist]
        rows = [5, 4, 3, 2, 1, 0] if step % 2 else range(6)  # any row order: groups of rows are what is wanted together
        base = [r for r in rows]
        parent, token, new = paged.eval_batch_beam([last[r] for r in base], base, [length[r] for r in base], scores[base], beams, beams)
        logits = np.stack([np.asarray(flat_logits(flat, toks[r // beams], hist[r])) for r in base]).astype(np.float64)
        lp = logits - np.log(np.exp(logits - logits.max(-1, keepdims=True)).sum(-1, keepdims=True)) - logits.max(-1, keepdims=True)
        total = scores[base][:, None] + lp
        tol = 2 * REL_TOL * np.abs(logits).max()
        picked = {}
        for g in range(2):
            part = total[g * beams:(g + 1) * beams]
            best = np.sort(part.ravel())[::-1][:beams]
            assert np.abs(new[g] - best).max() <= tol * (step + 1)
            for b in range(beams):
                assert parent[g, b] // beams == g
                assert abs(total[parent[g, b], token[g, b]] - new[g, b]) <= tol * (step + 1)
                picked[base[g * beams + b]] = (base[parent[g, b]], int(token[g, b]), new[g, b])
        paged.reorder(list(picked), [v[0] for v in picked.values()])
        hist = [hist[picked[r][0]] + [picked[r][1]] for r in range(6)]
        scores = np.array([picked[r][2] for r in range(6)])


def flat_logits(model, toks, more):
    return model.eval(np.concatenate([toks, more]), 0)


def test_beams_on_the_contiguous_cache(models):
    """The selection needs no pages: one step over rows of a contiguous model, with and without `want`."""
    spec, make, flat = models
    rng = np.random.default_rng(10)
    toks = rng.integers(0, spec.n_vocab, 4)
    for s in range(4):
        prompt(flat, s, rng.integers(0, spec.n_vocab, 5))
    logits = flat.eval_batch(toks, range(4), [5] * 4).astype(np.float64)
    m = logits.max(-1, keepdims=True)
    scores = np.array([-1.0, -2.0, -np.inf, -1.5])
    total = scores[:, None] + (logits - (m + np.log(np.exp(logits - m).sum(-1, keepdims=True))))
    parent, token, score = flat.eval_batch_beam(toks, range(4), [5] * 4, scores, 2, 4)
    for g in range(2):
        order = np.argsort(-total[2 * g:2 * g + 2].ravel(), kind="stable")[:4]
        assert (parent[g] == 2 * g + order // spec.n_vocab).all() and (token[g] == order % spec.n_vocab).all()
        # n exponentials and additions in double, three roundings of the score
        assert np.abs(score[g] - total[2 * g:2 * g + 2].ravel()[order]).max() <= (spec.n_vocab + 40) * 2.0 ** -52
    one = flat.eval_batch_beam(toks, range(4), [5] * 4, [0.0], 1, 2, np.array([0, 0, 1, 0]))
    assert (one[0] == 0).all() and (one[1][0] == np.argsort(-logits[2], kind="stable")[:2]).all()


def test_pages_run_out(models):
    spec, make, _ = models
    paged = make(pages=(16, 3, e.KV_F16))
    rng = np.random.default_rng(11)
    toks = rng.integers(0, spec.n_vocab, 32)
    prompt(paged, 0, toks[:16])
    prompt(paged, 1, toks[:20])
    with pytest.raises(MemoryError):
        prompt(paged, 2, toks[:1])
    with pytest.raises(MemoryError):
        paged.reorder([3, 2], [1, 1])
    assert paged.free_pages() == 0
    after = paged.eval_batch(toks[:1], [1], [20])[0]  # nothing was lost
    assert np.isfinite(after).all()
    paged.drop(0)
    prompt(paged, 2, toks[:1])


def test_refusals(models):
    spec, make, flat = models
    for pages in ((24, 4, 1), (16, 0, 1), (16, 4, 5)):
        with pytest.raises(ValueError):
            make(pages=pages)
    for call in (lambda: flat.reorder([0], [1]), lambda: flat.drop(0), flat.free_pages):
        with pytest.raises(e.ElbError):
            call()
    paged = make(pages=(16, 4, 1))
    for bad in (([0], [6]), ([-1], [0]), ([6], [0])):
        with pytest.raises(IndexError):
            paged.reorder(*bad)
    with pytest.raises(ValueError):
        paged.reorder([1, 1], [0, 2])
    with pytest.raises(IndexError):
        paged.drop(6)
    with pytest.raises(IndexError):
        paged.eval_batch([1], [0], [1])  # position 0 is missing
    beam = lambda scores=(0.0, 0.0), beams=2, k=2: flat.eval_batch_beam([1, 2], [0, 1], [0, 0], scores, beams, k)
    for kw in (dict(scores=(0.0,)), dict(beams=0), dict(beams=3), dict(k=0), dict(k=65)):
        with pytest.raises(ValueError):
            beam(**kw)
    beam()


def test_pages_that_the_rows_themselves_give_back(models):
    """A full pool: a sequence that starts over, and one that shares the last page of another, need only what they do not free."""
    spec, make, flat = models
    rng = np.random.default_rng(21)
    paged = make(pages=(16, 4, e.KV_PAIR))
    a, b = rng.integers(0, spec.n_vocab, 32), rng.integers(0, spec.n_vocab, 32)
    for s in (0, 1):  # two pages each: none is left
        assert rel(prompt(paged, s, a), prompt(flat, s, a)) <= REL_TOL
    assert paged.free_pages() == 0
    assert rel(prompt(paged, 0, b), prompt(flat, 0, b)) <= REL_TOL  # from position 0 on, over its own pages
    # both at once: one gives back a page that the other takes
    toks, seq = np.concatenate([b[:8], a[:16]]), [0] * 8 + [1] * 16
    pos, want = list(range(8)) + list(range(32, 48)), np.array([0] * 7 + [1] + [0] * 15 + [1], np.uint8)
    assert rel(paged.eval_batch(toks, seq, pos, want), flat.eval_batch(toks, seq, pos, want)) <= REL_TOL
    assert paged.free_pages() == 0
    # the sixth sequence goes on from the first, whose 8 rows fill half a page: no page for the copy; a full page is shared
    with pytest.raises(MemoryError):
        paged.reorder([5], [0])
    paged.drop(1)
    prompt(paged, 0, b[:16])
    paged.reorder([5], [0])
    assert paged.free_pages() == 3
    for s in (2, 3):
        prompt(paged, s, a[:16])
    assert paged.free_pages() == 1
    # both write from position 8 of the page they share: one copy, the other keeps the page
    prompt(flat, 0, b[:16])
    prompt(flat, 5, b[:16])
    toks, seq, pos = np.concatenate([a[:4], b[20:24]]), [0] * 4 + [5] * 4, list(range(8, 12)) * 2
    want = np.array([0, 0, 0, 1] * 2, np.uint8)
    assert rel(paged.eval_batch(toks, seq, pos, want), flat.eval_batch(toks, seq, pos, want)) <= REL_TOL
    assert paged.free_pages() == 0
