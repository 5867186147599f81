"""Handles of the paged cache and of rotary positions: ready for any stream when they are created."""
import pytest
import torch

import exactinfer_b200 as e
import test_gpu_kv as base

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
