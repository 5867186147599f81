"""Attention over the pages at the ends of the numbers' range: scores of any size."""
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
