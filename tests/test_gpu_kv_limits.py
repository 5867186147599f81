"""Paged cache, rotary positions and selection at the limits of what their calls allow: first calls under capture, huge logits,
results in place, spare pages that do not exist, expectations far off."""
import math
import subprocess
import sys

import numpy as np
import pytest
import torch

import exactinfer_b200 as e
import test_gpu_kv as base

pytestmark = pytest.mark.gpu
D, F64 = 128, torch.float64

FIRST_CALLS = """
import math, torch, exactinfer_b200 as e
x = torch.zeros(1, device="cuda")
rope, kv = e.Rope(128), e.KvCache(1, 2, 16, 64, %d)
i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
n, h = %d, 4
start, length, table = i32(0, n), i32(n + 5), torch.arange(16, dtype=torch.int32, device="cuda")
b = e.KvBatch(1, n, n, 256, start, length, table, 16)
q, k, v = (torch.randn(n, w * 128, device="cuda") for w in (h, 2, 2))
out, turned = torch.zeros_like(q), torch.zeros_like(q)
logits, scores = torch.randn(2, 5000, device="cuda"), torch.zeros(2, dtype=torch.float64, device="cuda")
parent, token, score = i32(0, 0), i32(0, 0), torch.zeros(2, dtype=torch.float64, device="cuda")
work = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
state = [torch.zeros(16, dtype=torch.int32, device="cuda") for _ in range(3)]

def calls():
    s = torch.cuda.current_stream().cuda_stream
    kv.append(0, b, k, v, 256, 256, rope, q=q, ldq=512, n_head=h, q_out=turned, ldqo=512, stream=s)
    kv.attention(0, b, turned, out, h, 0.1, work, work.numel(), stream=s)
    e.beam_select(logits, 5000, 1, 2, scores, 2, parent, token, score, work, work.numel(), stream=s)
    kv.reorder(1, i0, length, table, 16, spare, state[0], state[1], state[2], stream=s)

i0, spare = i32(0), i32(40)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    calls()
g.replay()
torch.cuda.synchronize()
got = [t.clone() for t in (out, token, score, *state)]
out.zero_(); token.zero_(); score.zero_()
calls()
torch.cuda.synchronize()
assert all(torch.equal(a, t) for a, t in zip(got, (out, token, score, *state)))
assert out.abs().sum() > 0 and torch.isfinite(score).all()
print("same")
"""


@pytest.mark.parametrize("kind,n", ((e.KV_F16, 1), (e.KV_PAIR, 40)))
def test_the_first_calls_of_a_process_are_captured(kind, n):
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS % (kind, n)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("size", (3e7, 3e8, 1e10, 2e10, 1e12))
def test_select_logits_whose_neighbours_are_far_apart(size):
    """fp32 numbers of this size are 2 to 65536 apart: the largest logit is the whole sum, and no term may be garbage."""
    x = base.randn(base.gen(40), 6, 7001) * size
    x[1] = x[1].abs()
    x[2] = -x[2].abs()
    x[3, ::3] = -math.inf
    scores = torch.linspace(-3, 0, 6, dtype=F64, device="cuda")
    base.agree(base.select(x, scores, 2, 3, 6), base.selected(x, scores, 2, 3, 6), 7001)


def test_select_scores_in_place():
    groups, beams, v = 5, 4, 3000
    x = base.randn(base.gen(41), groups * beams, v)
    scores = torch.randn(groups * beams, generator=base.gen(42), device="cuda", dtype=F64)
    want = base.select(x, scores, groups, beams, beams)
    parent, token = (torch.zeros(groups, beams, dtype=torch.int32, device="cuda") for _ in range(2))
    work = torch.empty(e.beam_select_work(v, groups, beams, 8), dtype=torch.uint8, device="cuda")
    call = lambda k, score, parent=parent: e.beam_select(x, v, groups, beams, scores, k, parent, token, score, work, work.numel(), stream=base.stream())
    for bad in (dict(k=3, score=scores), dict(k=4, score=scores.data_ptr() + 8), dict(k=4, score=torch.zeros(20, dtype=F64, device="cuda"), parent=scores)):
        with pytest.raises(ValueError):
            call(**bad)
    call(beams, scores)
    assert np.array_equal(parent.cpu().numpy(), want[0]) and np.array_equal(token.cpu().numpy(), want[1])
    assert np.array_equal(scores.cpu().numpy().reshape(groups, beams), want[2])


@pytest.mark.parametrize("spare", (-1, 6, 2**31 - 1))
def test_reorder_spare_pages_outside_the_pool(spare):
    """The second child of a row gets no copy, and not the first child's page either."""
    pool = torch.randn((2, 6, 2, 1, 1, 16, D), generator=base.gen(43), device="cuda").half()
    kv, before = e.KvCache(2, 1, 16, 6, 1, mem=pool), pool.clone()
    dev = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    lo, to, tk = (torch.full((n,), 9, dtype=torch.int32, device="cuda") for n in (3, 6, 3))
    kv.reorder(3, dev(1, 1, 1), dev(5, 20, 3), dev(0, -1, 1, 2, 3, -1), 2, dev(4, spare, 5), lo, to, tk, stream=base.stream())
    assert lo.tolist() == [20, 20, 20] and to.tolist() == [1, 2, 1, spare, 1, 5] and tk.tolist() == [0, 0, 1]
    before[:, 5] = before[:, 2]
    assert torch.equal(pool.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("nq", (1, 40))
@pytest.mark.parametrize("max_len", (0, 1, 2**31 - 1))
@pytest.mark.parametrize("max_q", (0, 2**31 - 1))
def test_attention_expectations_at_the_ends_of_their_range(nq, max_len, max_q):
    p = base.Paged(44, 2, 16, e.KV_PAIR, (nq, nq, nq), (nq, 300, 41)).fill()
    q, out = base.randn(p.g, p.n_tok, 4 * D), torch.full((p.n_tok, 4 * D), 7.0, device="cuda")
    b = e.KvBatch(3, p.n_tok, max_q, max_len, p.d_start, p.d_len, p.d_table, p.width)
    work = torch.empty(p.kv.attention_work(b, 4), dtype=torch.uint8, device="cuda")
    p.kv.attention(1, b, q, out, 4, 1 / math.sqrt(D), work, work.numel(), stream=base.stream())
    want, tol = p.expected(4, q)
    assert ((out.to(F64) - want).abs() <= tol).all()


def test_tables_longer_than_any_pool_are_refused():
    p = base.Paged(45, 2, 16, 1, (2,), (10,)).fill()
    q = torch.zeros(2, 4 * D, device="cuda")
    for ld, fits in ((2**30 // 16, True), (2**30 // 16 + 1, False)):
        b = e.KvBatch(1, 2, 2, 10, p.d_start, p.d_len, p.d_table, ld)
        work = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
        if fits:
            p.kv.attention(1, b, q, torch.empty_like(q), 4, 1.0, work, work.numel(), stream=base.stream())
        else:
            with pytest.raises(e.ElbError):
                p.kv.attention(1, b, q, torch.empty_like(q), 4, 1.0, work, work.numel(), stream=base.stream())
