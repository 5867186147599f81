"""Handles of the paged cache and of rotary positions: ready for any stream when they are created, errors of their own, what their calls
refuse."""
import pytest
import torch

import exactinfer_b200 as e
import test_gpu_kv as base
from exactinfer_b200 import capi

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("pages", (4, 1 << 18))  # 128 KB; 8 GB, whose zeroing takes milliseconds
def test_a_new_cache_is_used_at_once_on_another_stream(pages):
    """What the first call writes stays: the pool is zeroed, and the angles are there, when the create calls return."""
    side = torch.cuda.Stream()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    start, length, table, pos = i32(0, 1), i32(1), i32(pages - 1), i32(1000)
    x = base.randn(base.gen(60), 1, 6 * D)
    q, out, again, turned = torch.empty(1, 2 * D, device="cuda"), torch.empty(1, 2 * D, device="cuda"), torch.empty(1, 2 * D, device="cuda"), torch.empty(1, 2 * D, device="cuda")
    work = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    b = e.KvBatch(1, 1, 1, 1, start, length, table, 1)
    torch.cuda.synchronize()
    s, a = side.cuda_stream, x.data_ptr()
    for _ in range(3):
        kv = e.KvCache(1, 2, 16, pages, e.KV_PAIR)
        rope = e.Rope(D)
        rope.apply(x, pos, turned, 1, 2, ldx=6 * D, stream=s)
        kv.append(0, b, a + 8 * D, a + 16 * D, 6 * D, 6 * D, rope=rope, q=a, ldq=6 * D, n_head=2, q_out=q, ldqo=2 * D, stream=s)
        kv.attention(0, b, q, out, 2, 0.1, work, work.numel(), stream=s)
        torch.cuda.synchronize()
        kv.attention(0, b, q, again, 2, 0.1, work, work.numel(), stream=s)
        torch.cuda.synchronize()
        v = x[:, 4 * D:]  # one key: the result is its value
        assert ((again - v).abs() <= 2.0 ** -20 * v.abs() + 2.0 ** -24).all() and torch.equal(out, again)
        want, tol = base.turned(x[:, :2 * D].double().view(1, 2, D), pos, rope.config)
        assert ((turned.double().view(1, 2, D) - want).abs() <= tol).all()
        kv.close()


def test_working_memory_of_an_empty_batch_and_of_bad_ones():
    """No rows or no sequences: nothing to plan for, and the call does nothing with that much memory. What the call refuses needs 0 bytes."""
    kv = e.KvCache(1, 2, 16, 4)
    t = torch.zeros(16, dtype=torch.int32, device="cuda")
    batch = lambda **kw: e.KvBatch(**(dict(n_seq=2, n_tok=2, max_q=1, max_len=10, q_start=t, length=t, table=t, table_ld=2) | kw))
    work = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    q = torch.zeros(2, 4 * D, device="cuda")
    for kw in (dict(n_seq=0), dict(n_tok=0), dict(n_seq=0, n_tok=0, max_q=0, max_len=0, q_start=None, length=None, table=None, table_ld=0)):
        need = kv.attention_work(batch(**kw), 4)
        assert 0 < need <= work.numel()
        kv.attention(0, batch(**kw), q, q, 4, 1.0, work, need, stream=base.stream())
    for kw in (dict(n_seq=-1), dict(n_seq=65537), dict(n_tok=-1), dict(max_q=-1), dict(max_len=-1), dict(table_ld=-1), dict(table_ld=0), dict(table_ld=1 << 40)):
        assert kv.attention_work(batch(**kw), 4) == 0
    for h in (0, -2, 3, 2 * 65):
        assert kv.attention_work(batch(), h) == 0
    assert kv.attention_work(batch(), 2 * 64) > 0


@pytest.mark.parametrize("nq", (1, 40))
def test_a_wait_that_ran_out_is_reported_on_its_own_cache(nq):
    """The next attention call on that cache is refused, once; another cache's calls go on as if nothing had happened."""
    a, b = (base.Paged(61 + i, 2, 16, 1, (nq,), (50,)).fill() for i in range(2))
    qa, qb = base.randn(a.g, nq, 4 * D), base.randn(b.g, nq, 4 * D)
    want = a.attention(4, qa), b.attention(4, qb)
    for _ in range(2):
        assert capi.lib().elb_selftest_kv_wait_expiry(a.kv._h) == capi.OK
        assert torch.equal(b.attention(4, qb), want[1])
        with pytest.raises(e.ElbError, match="wait"):
            a.attention(4, qa)
        assert torch.equal(a.attention(4, qa), want[0])
    assert capi.lib().elb_selftest_kv_wait_expiry(None) == capi.ERR_INVALID


def test_results_that_overlap_what_they_are_made_from_are_refused():
    """Shared memory in any row, whatever the distance; columns of one buffer and neighbouring buffers are told apart from it."""
    buf = base.randn(base.gen(64), 40, 12 * D)
    at = lambda floats: buf.data_ptr() + 4 * floats
    ld, n = 12 * D, 8
    t = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    rope, pos, kv = e.Rope(D), torch.arange(n, device="cuda", dtype=torch.int32), e.KvCache(1, 2, 16, 4)
    b = e.KvBatch(1, n, n, n, t(0, n), t(n), t(0, 1), 2)
    work = torch.empty(kv.attention_work(b, 4), dtype=torch.uint8, device="cuda")
    turn = lambda x, y, ldx=ld, ldy=ld, rows=n: rope.apply(at(x), pos, at(y), rows, 4, ldx=ldx, ldy=ldy)
    attend = lambda x, y, ldx=ld, ldy=ld: kv.attention(0, b, at(x), at(y), 4, 0.1, work, work.numel(), ldq=ldx, ldo=ldy)
    append = lambda q, out, k, v, ldo=ld: kv.append(0, b, at(k), at(v), ld, ld, q=at(q), ldq=ld, n_head=4, q_out=at(out), ldqo=ldo)
    apart = [(0, 4 * D), (4 * D, 0), (8 * D, 0), (0, 7 * ld + 4 * D), (0, 8 * ld), (8 * ld, 0), (5 * ld + 4 * D, 0)]  # (4 heads are 4 D floats)
    for x, y in apart:
        turn(x, y)
        attend(x, y)
    meet = [(0, D), (D, 0), (0, 4), (0, 4 * D - 4), (0, 7 * ld), (7 * ld + 3 * D, 0), (2 * ld, ld + 9 * D), (ld + 9 * D, 0), (0, 3 * ld - 2 * D)]
    for x, y in meet:
        with pytest.raises(ValueError, match="overlap"):
            turn(x, y)
        with pytest.raises(ValueError, match="overlap"):
            attend(x, y)
        with pytest.raises(ValueError, match="overlap"):
            append(x, y, 16 * ld, 24 * ld)
        for k, v in ((y + 2 * D, 16 * ld), (16 * ld, y + D)):  # (keys and values are 2 D floats)
            with pytest.raises(ValueError, match="overlap"):
                append(30 * ld, y, k, v)
    with pytest.raises(ValueError, match="overlap"):
        attend(0, 0)
    with pytest.raises(ValueError, match="overlap"):
        turn(0, 2 * D, ldx=ld, ldy=4 * D, rows=1)
    turn(0, 0)
    append(0, 0, 4 * D, 6 * D)
    append(0, 8 * D, 4 * D, 6 * D)
    torch.cuda.synchronize()
