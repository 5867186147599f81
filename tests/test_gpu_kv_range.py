"""Attention over the pages and beam search's selection at the ends of the numbers' range: scores of any size, values that are not finite,
zeros of both signs."""
import math

import pytest
import torch

import exactinfer_b200 as e
import test_gpu_kv as base

pytestmark = pytest.mark.gpu
D, U, F64 = 128, 2.0 ** -24, torch.float64


@pytest.mark.parametrize("kind", (e.KV_F16, e.KV_PAIR))
@pytest.mark.parametrize("nq,n,h,hkv", [((1,), (300,), 4, 2), ((1,), (5000,), 2, 1), ((3, 1, 2), (70, 41, 700), 8, 2), ((40,), (300,), 4, 2),
                                        ((150, 33), (150, 2100), 6, 2)])
@pytest.mark.parametrize("size,scale", [(2.0 ** 21, 1.0), (2.0 ** 22, -1.0), (2.0 ** 24, 0.7), (2.0 ** 29, 1.0), (2.0 ** 40, 1.0), (2.0 ** 100, 1.0),
                                        (2.0 ** 90, 2.0 ** 90)])
def test_scores_of_any_size(nq, n, h, hkv, size, scale, kind):
    """Queries and keys are finite, so every row is finite; where one key is ahead of all others by more than the scores are off by, the
    row is that key's value. (Scores up to 2^186, beyond fp32: products are formed with scaled queries.)"""
    p = base.Paged(50, hkv, 32, kind, nq, n).fill()
    q = base.randn(p.g, p.n_tok, h * D) * size
    got = p.attention(h, q, scale=scale).to(F64)
    decided = rows = 0
    for s, (m, length) in enumerate(zip(nq, n)):
        r = slice(p.start[s], p.start[s] + m)
        see = torch.arange(length, device="cuda")[None] <= torch.arange(length - m, length, device="cuda")[:, None]
        for i in range(h):
            k, v = p.vals[s][:, i // (h // hkv)]
            x = q[r, i * D:(i + 1) * D].to(F64)
            raw = torch.where(see, (x @ k.T) * scale, -math.inf)
            off = ((x.abs() @ k.abs().T) * abs(scale) * see).amax(-1) * 28 * 2.0 ** -23  # of a score, as counted in base.Paged.expected
            best, at = raw.max(-1)
            second = raw.scatter(1, at[:, None], -math.inf).amax(-1)
            alone = best - second > 2 * off + 40  # every other weight is below e^-40
            mine = got[r, i * D:(i + 1) * D]
            most = v.abs().amax()
            # the weight as hi + lo (2^-22), the sum of two products, the quotient; the others' share
            tol = v[at].abs() * (2.0 ** -22 + 6 * U) + length * math.exp(-40) * most
            assert mine.isfinite().all() and (mine.abs() <= most * (1 + 2.0 ** -10)).all()
            assert ((mine - v[at]).abs() <= tol)[alone].all()
            decided, rows = decided + int(alone.sum()), rows + m
    assert decided > rows // 2


INF, NAN = math.inf, math.nan


@pytest.mark.parametrize("kind", (e.KV_F16, e.KV_PAIR))
@pytest.mark.parametrize("scale", (0.09, 30.0))
@pytest.mark.parametrize("nq,n,h,hkv,page", [(1, 90, 4, 2, 16), (1, 4000, 2, 1, 64), (4, 90, 4, 2, 16), (4, 3000, 8, 4, 128), (50, 90, 4, 2, 32), (200, 700, 2, 2, 256),
                                             (60, 5000, 4, 2, 16)])
def test_attended_values_that_are_not_finite(nq, n, h, hkv, page, scale, kind):
    """Every weight is above 0, so an infinite value is the result of its dimension in all rows that attend to it, wherever in a tile it lies
    and however little it weighs; infinities of both signs, or a NaN, give NaN. Other dimensions and earlier rows do not notice."""
    p = base.Paged(51, hkv, page, kind, (nq,), (n,)).fill()
    # (position, dimension, value), in the last key head
    places = [(0, 3, INF), (n - 1, 7, -INF), (n - nq // 2 - 1, 64, INF), (n // 3, 127, INF), (n // 2, 127, -INF), (n // 4, 90, NAN), (n // 5, 90, INF),
              (n - 2, 31, NAN), (n // 2 + 1, 0, -INF), (n // 2 + 2, 0, -INF)]
    v = p.vals[0][1, hkv - 1]
    for t, d, x in places:
        p.pool[1, int(p.table[0, t // page]), 1, hkv - 1, 0, t % page, d] = x
        if kind == e.KV_PAIR:
            p.pool[1, int(p.table[0, t // page]), 1, hkv - 1, 1, t % page, d] = 0.0
        v[t, d] = x
    q = base.randn(p.g, nq, h * D)
    got = p.attention(h, q, scale=scale).to(F64)
    want, tol = p.expected(h, q, scale)
    last = torch.arange(n - nq, n, device="cuda")
    for d in {d for _, d, _ in places}:
        odd = torch.zeros(nq, dtype=F64, device="cuda")
        for t, dd, x in places:
            if dd == d:
                odd += torch.where(last >= t, x, 0.0)
        for i in range(h - h // hkv, h):
            rows = odd != 0
            want[rows, i * D + d], tol[rows, i * D + d] = odd[rows], 0.0
    fine = want.isfinite()
    assert ((got - want).abs() <= tol)[fine].all()
    assert torch.equal(got[~fine].nan_to_num(5.0, INF, -INF), want[~fine].nan_to_num(5.0, INF, -INF))


@pytest.mark.parametrize("v", (1, 5, 700, 9001, 1100000))
@pytest.mark.parametrize("masked", (False, True))
def test_zeros_of_both_signs_are_equal_logits(v, masked):
    """The lower token goes first, whichever sign its zero has; with few zeros at the top and with more than a block keeps."""
    g = base.gen(52)
    zero = torch.where(torch.rand(4, v, generator=g, device="cuda") < 0.5, -0.0, 0.0)
    x = torch.where(torch.rand(4, v, generator=g, device="cuda") < 0.01, zero, -1.0)
    x[1], x[2, :-1] = zero[1], -2.0
    x[2, -1] = -0.0
    x[3] = -zero[1]
    allowed = torch.rand(4, v, generator=g, device="cuda") < 0.6 if masked else None
    scores = torch.tensor([-1.0, -1.0, -2.0, -2.0], dtype=F64, device="cuda")
    for k in (1, 2, 40):
        if k <= 2 * v:
            base.agree(base.select(x, scores, 2, 2, k, allowed), base.selected(x, scores, 2, 2, k, allowed), v)


@pytest.mark.parametrize("v", (2, 3, 5, 17, 64))
@pytest.mark.parametrize("size", (0.5, 3.0, 40.0))
def test_scores_of_small_vocabularies(v, size):
    """Few terms in a sum: every exponential counts with its own error, 11 * 2^-52 at most, and the additions with n 2^-53 on either side.
    Then each side rounds, by 2^-53 of the number: log-sum-exp (at most max |x| + ln v), logit less it (at most |want| + |score|) and the
    score (|want|); the scores are below 4, ln v below 5."""
    g = base.gen(53)
    x = base.randn(g, 2000, v) * size
    scores = torch.randn(2000, generator=g, device="cuda", dtype=F64)
    got, want = base.select(x, scores, 500, 4, 4), base.selected(x, scores, 500, 4, 4)
    assert (got[0] == want[0]).all() and (got[1] == want[1]).all()
    assert (abs(got[2] - want[2]) <= (11 + v + 8 + float(x.abs().max()) + 9 + 2 * abs(want[2])) * 2.0 ** -52).all()
