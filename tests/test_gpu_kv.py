"""The operators around the paged cache against plain formulas in 64 bits: rotary positions, append, attention over the pages, the
reordering of states and beam search's selection. Tolerances count roundings (u = 2^-24, half a step of fp32; fp16: 2^-11 relative
and 2^-25 absolute)."""
import math

import numpy as np
import pytest
import torch

import exactinfer_b200 as e

pytestmark = pytest.mark.gpu
D, U = 128, 2.0 ** -24
F64 = torch.float64


@pytest.fixture(scope="module", autouse=True)
def device():
    ok, why = e.cuda_available()
    assert ok, f"CUDA path unavailable: {why}"


def stream():
    return torch.cuda.current_stream().cuda_stream


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


# ---------------------------------------------------------------- rotary positions

def turned(x, pos, cfg):
    """(rotation of x[n][heads][head_dim] in 64 bits, bound of an fp32 result's error)"""
    f, m = e.rope_frequencies(cfg)
    f = torch.tensor(f, device="cuda")
    a = pos.to(F64)[:, None] * f
    c, s = (a.cos() * m)[:, None], (a.sin() * m)[:, None]
    dim = cfg.dim
    i, j = (slice(0, dim // 2), slice(dim // 2, dim)) if cfg.layout == e.ROPE_HALF else (slice(0, dim, 2), slice(1, dim, 2))
    y, tol = x.clone(), torch.zeros_like(x)
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., i] * s + x[..., j] * c
    # cosine and sine rounded once with m (2 u), one product and the sum rounded (2 u); the angle itself: positions times a
    # frequency, both sides rounded in double (2^-52 of the angle each, once more for turns)
    off = m * (4 * U + 3 * 2.0 ** -52 * a.abs()[:, None])
    tol[..., i] = tol[..., j] = (x[..., i].abs() + x[..., j].abs()) * off
    return y, tol


def normed(x, w, eps):
    """Norm in 64 bits; an fp32 result is off by the factor's rounding and two products: 3 u (and the factor's own 2^-40)."""
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.to(F64)


@pytest.mark.parametrize("n,heads,hd,dim,layout,scaling,norm", [
    (1, 1, 128, 128, 0, 0, False), (3, 5, 128, 64, 1, 2, True), (2049, 3, 128, 128, 0, 3, True), (17, 16, 64, 64, 0, 1, False),
    (5, 2, 256, 248, 1, 0, True), (33, 7, 32, 8, 0, 2, False), (9, 9, 80, 80, 0, 0, True), (4, 1, 2, 2, 1, 0, False), (130, 11, 96, 50, 1, 3, True),
    (70, 3, 128, 6, 0, 0, False)])
def test_rope(n, heads, hd, dim, layout, scaling, norm):
    g = gen(n * 31 + heads)
    r = e.Rope(hd, dim=dim, layout=layout, scaling=scaling, factor=4.0, orig_ctx=4096.0)
    x, w = randn(g, n, heads * hd), randn(g, hd) * 0.1 + 1
    pos = torch.randint(0, 1000000, (n,), generator=g, device="cuda", dtype=torch.int32)
    pos[0] = 0 if n > 1 else 77
    y = torch.full_like(x, float("nan"))
    r.apply(x, pos, y, n, heads, norm=w if norm else None, eps=1e-6, stream=stream())
    x64 = x.to(F64).view(n, heads, hd)
    if norm:
        x64 = normed(x64, w, 1e-6)
    want, tol = turned(x64, pos, r.config)
    spread = want.abs() + tol / (4 * U)  # what a relative error of the rotated inputs grows to
    assert ((y.to(F64).view_as(want) - want).abs() <= tol + (4 * U * spread if norm else 0)).all()
    if not norm and dim < hd:
        assert torch.equal(y.view(n, heads, hd)[..., dim:], x.view(n, heads, hd)[..., dim:])


def test_rope_far_positions():
    g = gen(1)
    r = e.Rope(128)
    pos = torch.tensor([0, 1, 2**24 + 1, 2**31 - 1, -1, -2**31, 1000003], device="cuda", dtype=torch.int32)
    x = randn(g, 7, 2 * 128)
    y = torch.empty_like(x)
    r.apply(x, pos, y, 7, 2, stream=stream())
    want, tol = turned(x.to(F64).view(7, 2, 128), pos, r.config)
    assert ((y.to(F64).view_as(want) - want).abs() <= tol).all()
    assert torch.equal(y[0], x[0])


@pytest.mark.parametrize("off", (0, 1))
def test_rope_in_place_and_strides(off):
    """In place, rows further apart than their width, and (off = 1) rows that start on no 16-byte boundary."""
    g = gen(2)
    r = e.Rope(128, dim=96)
    buf = randn(g, 21 * 600 + 8)
    x = buf[off:off + 21 * 600].view(21, 600)
    before = buf.clone()
    pos = torch.arange(21, device="cuda", dtype=torch.int32) * 37
    r.apply(x, pos, x, 21, 4, ldx=600, ldy=600, stream=stream())
    old = before[off:off + 21 * 600].view(21, 600)
    want, tol = turned(old[:, :512].to(F64).view(21, 4, 128), pos, r.config)
    assert ((x[:, :512].to(F64).reshape(21, 4, 128) - want).abs() <= tol).all()
    assert torch.equal(x[:, 512:], old[:, 512:]) and torch.equal(buf[:off], before[:off]) and torch.equal(buf[off + 12600:], before[off + 12600:])


@pytest.mark.parametrize("size", (1e-25, 1e25))
def test_rope_norm_beyond_fp32_squares(size):
    r = e.Rope(64)
    x = randn(gen(3), 5, 64) * size
    y, w, pos = torch.empty_like(x), torch.ones(64, device="cuda"), torch.zeros(5, device="cuda", dtype=torch.int32)
    r.apply(x, pos, y, 5, 1, norm=w, eps=0.0, stream=stream())
    want = normed(x.to(F64), w, 0.0)
    assert ((y - want).abs() <= 4 * U * want.abs()).all()


def test_rope_norm_weights_anywhere():
    g = gen(40)
    r, x, w = e.Rope(128), randn(g, 5, 256), randn(g, 129) * 0.1 + 1
    y, pos = torch.empty_like(x), torch.arange(5, device="cuda", dtype=torch.int32)
    r.apply(x, pos, y, 5, 2, norm=w[1:], eps=1e-6, stream=stream())
    want, tol = turned(normed(x.to(F64).view(5, 2, 128), w[1:], 1e-6), pos, r.config)
    assert ((y.to(F64).view_as(want) - want).abs() <= tol + 4 * U * (want.abs() + tol / (4 * U))).all()


def test_rope_refusals():
    r, x, p = e.Rope(128), torch.zeros(4, 256, device="cuda"), torch.zeros(4, device="cuda", dtype=torch.int32)
    for kw in (dict(n=-1), dict(heads=0), dict(ldx=255), dict(ldy=100), dict(y=None), dict(x=None), dict(pos=None), dict(eps=-1.0, norm=x)):
        args = dict(x=x, pos=p, y=torch.zeros_like(x), n=4, heads=2) | kw
        with pytest.raises(ValueError):
            r.apply(**args)
    with pytest.raises(ValueError):
        r.apply(x, p, x, 4, 2, ldx=256, ldy=260)
    r.apply(None, None, None, 0, 2)  # no rows: nothing to do


# ---------------------------------------------------------------- a batch over a pool

class Paged:
    """Sequences with nq new rows and len positions in a pool whose pages lie in random order; unused values are NaN."""

    def __init__(self, seed, hkv, page, kind, nq, lens, layers=2, layer=1, extra_rows=0, gap=0, width=None):
        self.g = g = gen(seed)
        self.hkv, self.page, self.kind, self.nq, self.lens, self.layer = hkv, page, kind, list(nq), list(lens), layer
        counts = [(n + page - 1) // page for n in lens]
        pages = sum(counts) + 2
        self.width = width or max(max(counts), 1) + 1
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table = torch.full((len(lens), self.width), -1, dtype=torch.int32)
        at = 0
        for s, c in enumerate(counts):
            self.table[s, :c] = torch.tensor(order[at:at + c], dtype=torch.int32)
            at += c
        self.unused = order[at:]
        self.pool = torch.full((layers, pages, 2, hkv, kind, page, D), float("nan"), dtype=torch.half, device="cuda")
        self.start = [gap]
        for a in nq:
            self.start.append(self.start[-1] + a)
        self.n_tok = self.start[-1] + extra_rows
        dev = lambda x: torch.as_tensor(x, dtype=torch.int32).cuda()
        self.d_start, self.d_len, self.d_table = dev(self.start), dev(self.lens), dev(self.table)
        self.kv = e.KvCache(layers, hkv, page, pages, kind, mem=self.pool)
        self.batch = e.KvBatch(len(lens), self.n_tok, max(nq), max(0, *lens, 0), self.d_start, self.d_len, self.d_table, self.width)

    def fill(self, scale=1.0):
        """Random keys and values at every position of every sequence: [2][hkv][len][D] each, as stored."""
        self.vals = []
        for s, n in enumerate(self.lens):
            x = randn(self.g, 2, self.hkv, max(n, 0), D) * scale
            hi = x.half()
            planes = [hi] if self.kind == 1 else [hi, (x - hi.float()).half()]
            for p in range(n):
                pg = int(self.table[s, p // self.page])
                for i, pl in enumerate(planes):
                    self.pool[self.layer, pg, :, :, i, p % self.page] = pl[:, :, p]
            self.vals.append(sum(pl.to(F64) for pl in planes))
        return self

    def attention(self, h, q, out=None, scale=None, work=None, st=None):
        out = torch.full_like(q, float("nan")) if out is None else out
        need = self.kv.attention_work(self.batch, h)
        work = torch.empty(need, dtype=torch.uint8, device="cuda") if work is None else work
        self.kv.attention(self.layer, self.batch, q, out, h, 1 / math.sqrt(D) if scale is None else scale, work, work.numel(), ldq=q.stride(0),
                          ldo=out.stride(0), stream=stream() if st is None else st)
        return out

    def expected(self, h, q, scale=None):
        """(output, bound) of every row that belongs to a sequence, in 64 bits."""
        scale = 1 / math.sqrt(D) if scale is None else scale
        out, tol = torch.zeros(self.n_tok, h * D, dtype=F64, device="cuda"), torch.zeros(self.n_tok, h * D, dtype=F64, device="cuda")
        for s, (nq, n) in enumerate(zip(self.nq, self.lens)):
            for i in range(h if n else 0):
                k, v = self.vals[s][:, i // (h // self.hkv)]
                rows = slice(self.start[s], self.start[s] + nq)
                x = q[rows, i * D:(i + 1) * D].to(F64)
                see = torch.arange(n, device="cuda")[None] <= torch.arange(n - nq, n, device="cuda")[:, None]
                raw = (x @ k.T) * scale
                size = (x.abs() @ k.abs().T) * abs(scale)
                w = torch.where(see, raw, -math.inf).softmax(-1).nan_to_num(0.0)
                kn, vn = torch.where(k.isfinite(), k, 0), torch.where(v.isfinite(), v, 0)
                out[rows, i * D:(i + 1) * D] = w @ vn
                # a score: operands of 22 bits (2 * 2^-22), at most 24 additions truncated by 2^-23 each, two products; a weight
                # twice that (numerator and sum). Weights and values of 22 bits, 12 additions within a tile and a sum over
                # n / 64 tiles for output and denominator, the exponential's 2^-22 and a few roundings
                d = (size * see).amax(-1, keepdim=True).nan_to_num(0.0) * 28 * 2.0 ** -23
                tol[rows, i * D:(i + 1) * D] = (w @ vn.abs()) * (2 * d + (96 + n / 32) * U) + 2.0 ** -60
        return out, tol

    def rows(self):
        return torch.arange(self.start[0], self.start[-1], device="cuda")


def check(p, h, q=None, **kw):
    q = randn(p.g, p.n_tok, h * D) if q is None else q
    got = p.attention(h, q, **kw)
    want, tol = p.expected(h, q, kw.get("scale"))
    r = p.rows()
    off = (got[r].to(F64) - want[r]).abs()
    assert (off <= tol[r]).all(), f"off by {float((off - tol[r]).max()):.3g} more than allowed"
    return got


# ---------------------------------------------------------------- append

@pytest.mark.parametrize("hkv,h,page,kind,nq,lens", [
    (1, 1, 16, 1, (1,), (1,)), (8, 32, 16, 2, (1, 1, 1), (40, 17, 16)), (2, 6, 64, 2, (5, 70, 1), (5, 200, 65)), (8, 64, 128, 1, (300,), (300,)),
    (3, 3, 256, 2, (2, 2100), (2, 2500)), (4, 4, 32, 1, (4, 3), (2, 0))])
def test_append(hkv, h, page, kind, nq, lens):
    p = Paged(7, hkv, page, kind, nq, lens, extra_rows=2, gap=1)
    before = p.pool.clone()
    r = e.Rope(D, scaling=e.ROPE_YARN, factor=4.0, orig_ctx=1024.0)
    ld = (h + 2 * hkv) * D + 8
    qkv = randn(p.g, p.n_tok, ld)
    qn, kn = randn(p.g, D) * 0.1 + 1, randn(p.g, D) * 0.1 + 1
    qo = torch.full((p.n_tok, h * D + 4), 9.0, device="cuda")
    a = qkv.data_ptr()
    p.kv.append(p.layer, p.batch, a + 4 * h * D, a + 4 * (h + hkv) * D, ld, ld, rope=r, k_norm=kn, eps=1e-6, q=a, ldq=ld, n_head=h, q_norm=qn, q_out=qo,
                ldqo=h * D + 4, stream=stream())
    written = torch.zeros(p.pool.shape[1], page, dtype=torch.bool)
    touched = torch.zeros(p.n_tok, dtype=torch.bool)
    for s, (m, n) in enumerate(zip(nq, lens)):
        i0 = max(0, m - n)
        if i0 == m:
            continue
        rows = slice(p.start[s] + i0, p.start[s] + m)
        touched[rows] = True
        pos = torch.arange(n - m + i0, n, device="cuda")
        x = qkv[rows, :(h + 2 * hkv) * D].to(F64).view(-1, h + 2 * hkv, D)
        q, qt = turned(normed(x[:, :h], qn, 1e-6), pos, r.config)
        k, kt = turned(normed(x[:, h:h + hkv], kn, 1e-6), pos, r.config)
        assert ((qo[rows, :h * D].to(F64).view_as(q) - q).abs() <= qt + 4 * U * (q.abs() + qt / (4 * U))).all()
        for j, t in enumerate(pos.tolist()):
            pg = int(p.table[s, t // page])
            got = p.pool[p.layer, pg, :, :, :, t % page].to(F64).sum(2)  # [2][hkv][D]
            rel = 2.0 ** -11 if kind == 1 else 2.0 ** -22
            f32 = kt[j] + 4 * U * (k[j].abs() + kt[j] / (4 * U))
            assert ((got[0] - k[j]).abs() <= rel * k[j].abs() + 2 * f32 + 2.0 ** -25).all()
            v = x[j, h + hkv:]
            assert ((got[1] - v).abs() <= rel * v.abs() + 2.0 ** -25).all()
            written[pg, t % page] = True
    assert (qo[~touched.cuda()] == 9.0).all() and (qo[:, h * D:] == 9.0).all()
    keep = ~written.cuda()[None, :, None, None, None, :, None].expand_as(p.pool)
    keep[0] = True
    assert torch.equal(p.pool[keep].view(torch.int16), before[keep].view(torch.int16))  # everything else as it was


def test_append_without_rotation_in_place_and_infinite_values():
    p = Paged(8, 2, 16, 2, (3,), (20,))
    x = randn(p.g, 3, 8 * D)
    x[1, 6 * D] = float("inf")
    x[2, 4 * D + 5] = 1e6
    before = x.clone()
    a = x.data_ptr()
    p.kv.append(1, p.batch, a + 16 * D, a + 24 * D, 8 * D, 8 * D, q=a, ldq=8 * D, n_head=4, q_out=a, ldqo=8 * D, stream=stream())
    assert torch.equal(x, before)  # no norm, no positions: the queries are what they were
    got = p.pool[1, int(p.table[0, 1])][:, :, :, 1:4].float().sum(2)  # [2][2][3][D]
    want = before[:, 4 * D:].view(3, 2, 2, D).permute(1, 2, 0, 3)
    want = torch.where(want.abs() > 65520, want * float("inf"), want)  # beyond fp16's range
    fine = want.isfinite()
    assert torch.equal(got[~fine], want[~fine])
    assert ((got - want)[fine].abs() <= 2.0 ** -22 * want[fine].abs() + 2.0 ** -25).all()


@pytest.mark.parametrize("bad", (-1, 1 << 20, -2**31, 2**31 - 1))
def test_bad_pages_are_not_touched(bad):
    """A page outside the pool is not written by append and reads as zeros in attention."""
    p = Paged(9, 2, 16, 1, (1, 1), (33, 20)).fill()
    p.d_table[0, 1] = bad
    before = p.pool.clone()
    x = randn(p.g, 2, 4 * D)
    p.d_len[0] = 17 + 1  # the new token of sequence 0 falls into the bad page
    a = x.data_ptr()
    p.kv.append(1, p.batch, a, a + 8 * D, 4 * D, 4 * D, stream=stream())
    changed = (p.pool.view(torch.int16) != before.view(torch.int16)).flatten(2).any(-1).nonzero().tolist()
    assert changed == [[1, int(p.table[1, 1])]]
    p.pool.copy_(before)
    p.d_len[0] = 33
    q = randn(p.g, 2, 4 * D)
    p.vals[0][:, :, 16:32] = 0
    got, (want, tol) = p.attention(4, q), p.expected(4, q)
    assert ((got.to(F64) - want).abs() <= tol).all()


# ---------------------------------------------------------------- attention

ONE = [(1, 1, 16, (1,), (1,)), (8, 16, 16, (1,), (41,)), (8, 32, 32, (1,) * 5, (1, 15, 16, 17, 700)), (8, 64, 64, (1, 1), (2000, 64)),
       (2, 10, 128, (1, 1, 1), (129, 128, 5)), (1, 64, 256, (1,), (257,)), (4, 4, 16, (1,) * 33, tuple(range(1, 34))), (2, 14, 16, (2, 1, 4), (70, 300, 4))]
CHUNK = [(2, 8, 16, (2,), (2,)), (8, 16, 32, (3, 77, 20), (203, 400, 20)), (2, 2, 64, (130,), (130,)), (1, 5, 128, (65, 1), (65, 400)),
         (1, 7, 16, (100,), (163,)), (2, 16, 256, (33, 64, 31), (300, 64, 1000)), (1, 64, 64, (9,), (80,)), (4, 32, 16, (512,), (700,))]


@pytest.mark.parametrize("kind", (e.KV_F16, e.KV_PAIR))
@pytest.mark.parametrize("hkv,h,page,nq,lens", ONE + CHUNK)
def test_attention(hkv, h, page, nq, lens, kind):
    check(Paged(11, hkv, page, kind, nq, lens).fill(), h)


@pytest.mark.parametrize("kind", (e.KV_F16, e.KV_PAIR))
@pytest.mark.parametrize("nq,lens", [((3, 5, 2), (2, 0, 2)), ((1, 1), (0, 3)), ((40, 0, 30), (7, 9, 30)), ((70,), (-3,))])
def test_rows_without_keys_are_zero(nq, lens, kind):
    """More rows than positions (a padded front), no positions at all, a negative length, a sequence without rows."""
    p = Paged(12, 2, 16, kind, nq, lens).fill()
    h = 4
    q = randn(p.g, p.n_tok, h * D)
    lens0 = [max(n, 0) for n in lens]
    for s, (m, n) in enumerate(zip(nq, lens0)):
        q[p.start[s]:p.start[s] + max(m - n, 0)] = float("nan")  # nobody reads these
    got = p.attention(h, q)
    p.lens = lens0
    want, tol = p.expected(h, q.nan_to_num(0.0))
    assert ((got.to(F64) - want).abs() <= tol).all()
    for s, (m, n) in enumerate(zip(nq, lens0)):
        assert (got[p.start[s]:p.start[s] + max(m - n, 0)] == 0).all()


@pytest.mark.parametrize("nq", (1, 40))
def test_rows_outside_are_left_alone(nq):
    p = Paged(13, 2, 16, 1, (nq, nq), (50, 60), extra_rows=3, gap=2).fill()
    q = randn(p.g, p.n_tok, 8 * D + 4)
    out = torch.full((p.n_tok, 8 * D + 12), 5.0, device="cuda")
    p.attention(8, q, out=out)
    want, tol = p.expected(8, q)
    r = p.rows()
    assert ((out[r, :8 * D].to(F64) - want[r]).abs() <= tol[r]).all()
    assert (out[:2] == 5).all() and (out[-3:] == 5).all() and (out[:, 8 * D:] == 5).all()


@pytest.mark.parametrize("kind", (e.KV_F16, e.KV_PAIR))
@pytest.mark.parametrize("what", (float("nan"), float("inf"), -float("inf")))
@pytest.mark.parametrize("nq", (4, 50))
def test_masked_places_have_no_influence(nq, what, kind):
    """Behind the length everything is NaN already; here also keys and values that only the last two rows may see."""
    p = Paged(14, 2, 16, kind, (nq,), (90,)).fill()
    q = randn(p.g, nq, 4 * D)
    clean, tol = p.expected(4, q)
    t = 88
    p.pool[1, int(p.table[0, t // 16]), :, :, 0, t % 16] = what
    if kind == e.KV_PAIR:
        p.pool[1, int(p.table[0, t // 16]), :, :, 1, t % 16] = 0
    got = p.attention(4, q)
    assert ((got[:nq - 2].to(F64) - clean[:nq - 2]).abs() <= tol[:nq - 2]).all()
    if what != what:
        assert got[nq - 2:].isnan().all()


@pytest.mark.parametrize("kind", (e.KV_F16, e.KV_PAIR))
@pytest.mark.parametrize("nq,scale,size", [(1, 0.0, 1.0), (20, -0.1, 1.0), (1, 1.0, 3.0), (33, 1.0, 3.0), (40, 1e-3, 100.0), (1, 0.05, 1e-3), (30, 0.05, 1e-3)])
def test_scales_and_sizes(nq, scale, size, kind):
    """No scale, a negative one, scores so far apart that all weight is on few keys, large and small values."""
    p = Paged(15, 2, 32, kind, (nq,), (150,)).fill(size)
    check(p, 4, q=randn(p.g, nq, 4 * D) * (1e4 if size < 1 else 1.0), scale=scale)


@pytest.mark.parametrize("factor", (1e-20, 1e20))
@pytest.mark.parametrize("nq", (1, 40))
def test_queries_far_outside_fp16(nq, factor):
    p = Paged(16, 2, 32, e.KV_PAIR, (nq,), (100,)).fill()
    check(p, 8, q=randn(p.g, nq, 8 * D) * factor, scale=0.09 / factor)


@pytest.mark.parametrize("nq,n,h", [(1, 40000, 8), (5, 12345, 2), (130, 9000, 4)])
def test_long_contexts(nq, n, h):
    p = Paged(17, 1, 64, e.KV_F16, (nq,), (n,))
    x = randn(p.g, 2, 1, n, D).half()
    for i in range((n + 63) // 64):
        m = min(64, n - 64 * i)
        p.pool[1, int(p.table[0, i]), :, :, 0, :m] = x[:, :, 64 * i:64 * i + m]
    p.vals = [x.to(F64)]
    check(p, h)


def test_many_ragged_sequences():
    rng = np.random.default_rng(3)
    lens = rng.integers(1, 300, 200).tolist()
    nq = [int(rng.integers(0, min(n, 6) + 1)) for n in lens]
    nq[5] = min(lens[5], 3)
    check(Paged(18, 2, 16, e.KV_PAIR, nq, lens).fill(), 4)


@pytest.mark.parametrize("max_q,max_len", [(0, 0), (1, 1), (4096, 1 << 20)])
@pytest.mark.parametrize("nq", (1, 45))
def test_expectations_do_not_change_results(nq, max_q, max_len):
    """max_q and max_len choose kernels; the lengths on the device are what counts."""
    p = Paged(19, 2, 16, e.KV_F16, (nq, 2), (500, 300)).fill()
    p.batch = e.KvBatch(2, p.n_tok, max_q, max_len, p.d_start, p.d_len, p.d_table, p.width)
    check(p, 8)


@pytest.mark.parametrize("kind", (e.KV_F16, e.KV_PAIR))
@pytest.mark.parametrize("h,hkv", [(8, 2), (24, 2), (4, 4)])
@pytest.mark.parametrize("order", (0, 1))
def test_single_tokens_and_chunks_in_one_batch(order, h, hkv, kind):
    """A server's step: one token of most sequences, chunks of some, nothing of others, rows in front of and behind them all."""
    nq = [1, 1, 1, 40, 1, 0, 1, 9, 1, 4, 1, 1, 70, 1, 2, 1] + [1] * 40
    lens = [300, 5, 1, 700, 16, 33, 1200, 9, 64, 400, 17, 1, 70, 250, 1, 90] + list(range(1, 400, 10))
    if order:
        nq, lens = nq[::-1], lens[::-1]
    p = Paged(33, hkv, 16, kind, nq, lens, extra_rows=3, gap=2).fill()
    q = randn(p.g, p.n_tok, h * D)
    want, tol = p.expected(h, q)
    r = p.rows()
    for max_q, max_len in ((70, 1200), (1, 1200), (200, 1), (30, 5000)):
        p.batch = e.KvBatch(len(nq), p.n_tok, max_q, max_len, p.d_start, p.d_len, p.d_table, p.width)
        got = p.attention(h, q, out=torch.full_like(q, 7.0))
        assert ((got[r].to(F64) - want[r]).abs() <= tol[r]).all()
        assert (got[:2] == 7).all() and (got[-3:] == 7).all()


def test_lengths_beyond_the_table():
    """More positions than the table has pages for: nothing outside is read; the keys that there are count, with zeros behind."""
    p = Paged(20, 2, 16, 1, (1, 40), (48, 64), width=4).fill()
    p.d_len[0] = 1000
    q = randn(p.g, p.n_tok, 4 * D)
    got = p.attention(4, q)
    want, tol = p.expected(4, q)
    assert ((got[1:].to(F64) - want[1:]).abs() <= tol[1:]).all() and got[0].isfinite().all()


def test_same_bits_every_time_and_dirty_work():
    p = Paged(21, 8, 16, e.KV_F16, (1,) * 20, [int(n) for n in np.random.default_rng(1).integers(1, 3000, 20)]).fill()
    q = randn(p.g, 20, 32 * D)
    work = torch.full((p.kv.attention_work(p.batch, 32),), 255, dtype=torch.uint8, device="cuda")
    first = p.attention(32, q, work=work)
    for _ in range(3):
        assert torch.equal(p.attention(32, q, work=work), first)


@pytest.mark.parametrize("nq", (1, 50))
def test_captured_and_replayed_with_other_lengths(nq):
    """A captured call follows the lengths, tables and values that are there when it is replayed."""
    p = Paged(22, 2, 16, e.KV_F16, (nq, nq), (200, 300)).fill()
    q, out = randn(p.g, p.n_tok, 8 * D), torch.zeros(p.n_tok, 8 * D, device="cuda")
    work = torch.empty(p.kv.attention_work(p.batch, 8), dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p.attention(8, q, out=out, work=work)
    for lens in ((200, 300), (150, 64), (60, 299)):
        p.lens = list(lens)
        vals = p.vals
        p.vals = [v[:, :, :n] for v, n in zip(vals, lens)]
        p.d_len.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(randn(p.g, *q.shape))
        g.replay()
        want, tol = p.expected(8, q)
        assert ((out.to(F64) - want).abs() <= tol).all()
        p.vals = vals


def test_two_streams_at_once():
    a, b = Paged(23, 8, 16, 1, (1,) * 8, (900,) * 8).fill(), Paged(24, 8, 32, 2, (60, 30), (700, 90)).fill()
    qa, qb = randn(a.g, 8, 32 * D), randn(b.g, 90, 16 * D)
    wa, wb = a.attention(32, qa), b.attention(16, qb)
    oa, ob = torch.zeros_like(wa), torch.zeros_like(wb)
    work = [torch.empty(a.kv.attention_work(a.batch, 32), dtype=torch.uint8, device="cuda"),
            torch.empty(b.kv.attention_work(b.batch, 16), dtype=torch.uint8, device="cuda")]
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        a.attention(32, qa, out=oa, work=work[0], st=s.cuda_stream)
        b.attention(16, qb, out=ob, work=work[1], st=t.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(oa, wa) and torch.equal(ob, wb)


def test_attention_and_append_refusals():
    p = Paged(25, 2, 16, 1, (2,), (10,)).fill()
    q, out = torch.zeros(2, 4 * D, device="cuda"), torch.zeros(2, 4 * D, device="cuda")
    work = torch.empty(p.kv.attention_work(p.batch, 4) + 256, dtype=torch.uint8, device="cuda")
    w = work.numel() - 256

    def call(layer=1, batch=p.batch, q=q, out=out, h=4, scale=1.0, work=work, wb=w, ldq=4 * D, ldo=4 * D):
        p.kv.attention(layer, batch, q, out, h, scale, work, wb, ldq=ldq, ldo=ldo, stream=stream())

    call()
    bad = lambda **kw: e.KvBatch(**(dict(n_seq=1, n_tok=2, max_q=2, max_len=10, q_start=p.d_start, length=p.d_len, table=p.d_table, table_ld=p.width) | kw))
    for kw in (dict(q=None), dict(out=None), dict(h=3), dict(h=0), dict(h=2 * 65), dict(scale=float("nan")), dict(work=None), dict(wb=w - 1),
               dict(work=work.data_ptr() + 16), dict(ldq=4 * D - 4), dict(ldo=0), dict(batch=bad(n_seq=-1)), dict(batch=bad(n_tok=-1)),
               dict(batch=bad(q_start=None)), dict(batch=bad(length=None)), dict(batch=bad(table=None)), dict(batch=bad(table_ld=0)),
               dict(batch=bad(max_q=-1)), dict(batch=bad(max_len=-1))):
        with pytest.raises(ValueError):
            call(**kw)
    for layer in (-1, 2):
        with pytest.raises(IndexError):
            call(layer=layer)
    for kw in (dict(q=q.data_ptr() + 4), dict(out=out.data_ptr() + 8), dict(ldq=4 * D + 1), dict(batch=bad(n_seq=70000)), dict(batch=bad(table_ld=1 << 40))):
        with pytest.raises(e.ElbError):
            call(**kw)
    call(batch=bad(n_tok=0), q=None, out=None, work=None, wb=0)  # no rows, no sequences: nothing to do
    call(batch=bad(n_seq=0, q_start=None, length=None, table=None, table_ld=0))

    x = torch.zeros(2, 8 * D, device="cuda")
    rope = e.Rope(D)

    def app(layer=1, k=x, v=x, ldk=8 * D, ldv=8 * D, **kw):
        p.kv.append(layer, p.batch, k, v, ldk, ldv, stream=stream(), **kw)

    for kw in (dict(k=None), dict(v=None), dict(ldk=D), dict(ldv=0), dict(q=x, ldq=8 * D, n_head=0, q_out=x, ldqo=8 * D), dict(q=x, ldq=8 * D, n_head=4),
               dict(q=x, ldq=8 * D, n_head=4, q_out=x, ldqo=8 * D + 4), dict(q=x, ldq=100, n_head=4, q_out=out, ldqo=4 * D), dict(k_norm=x, eps=-1.0),
               dict(rope=e.Rope(64))):
        with pytest.raises(ValueError):
            app(**kw)
    for kw in (dict(k=x.data_ptr() + 4), dict(ldv=8 * D + 2), dict(rope=e.Rope(D, dim=6)), dict(k_norm=x.data_ptr() + 4)):
        with pytest.raises(e.ElbError):
            app(**kw)
    with pytest.raises(IndexError):
        app(layer=5)
    app(rope=rope)


# ---------------------------------------------------------------- states of a beam search

@pytest.mark.parametrize("kind,page,layers", [(1, 16, 3), (2, 64, 1), (1, 256, 2)])
@pytest.mark.parametrize("parents", [(0,), (0, 0, 0, 0), (3, 2, 1, 0), (1, 1, -1, 7), (2, 2, 3, 3)])
def test_reorder(parents, kind, page, layers):
    n = len(parents)
    lens = [page * 2 + 5, page, 1, 3 * page + 1][:n]
    g = gen(26)
    counts = [(x + page - 1) // page for x in lens]
    pages, width = sum(counts) + n + 1, max(counts) + 2
    pool = torch.randn((layers, pages, 2, 3, kind, page, D), generator=g, device="cuda").half()
    order = torch.randperm(pages).tolist()
    table, at = torch.full((n, width), -1, dtype=torch.int32), 0
    for r, c in enumerate(counts):
        table[r, :c] = torch.tensor(order[at:at + c], dtype=torch.int32)
        at += c
    table[0, counts[0]] = order[-1]  # a page reserved ahead, behind the length
    spare = torch.tensor(order[at:at + n], dtype=torch.int32)
    kv = e.KvCache(layers, 3, page, pages, kind, mem=pool)
    before = pool.clone()
    want = before.clone()
    wt, wl, wk, seen = torch.full_like(table, -1), [0] * n, [0] * n, set()
    for r, q in enumerate(parents):
        if not 0 <= q < n:
            continue
        wl[r] = lens[q]
        wt[r, :counts[q]] = table[q, :counts[q]]
        if lens[q] % page and q in seen:
            want[:, spare[r].long()] = before[:, table[q, counts[q] - 1].long()]
            wt[r, counts[q] - 1], wk[r] = spare[r], 1
        seen.add(q)
    dev = lambda x: torch.as_tensor(x, dtype=torch.int32).cuda()
    lo, to, tk = (torch.full(s, 99, dtype=torch.int32, device="cuda") for s in ((n,), (n, width), (n,)))
    kv.reorder(n, dev(parents), dev(lens), dev(table), width, dev(spare), lo, to, tk, stream=stream())
    assert to.tolist() == wt.tolist() and lo.tolist() == wl and tk.tolist() == wk
    assert torch.equal(pool.view(torch.int16), want.view(torch.int16))


def test_reorder_many_rows_and_bad_pages():
    n, page, layers = 700, 16, 2
    pool = torch.randn((layers, 2 * n, 2, 1, 1, page, D), generator=gen(27), device="cuda").half()
    kv = e.KvCache(layers, 1, page, 2 * n, 1, mem=pool)
    rng = np.random.default_rng(2)
    parent = rng.integers(-2, n + 2, n)
    lens = rng.integers(0, page + 1, n)
    dev = lambda x: torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()
    table, spare = np.arange(n)[:, None], n + np.arange(n)
    bad = int(np.bincount(parent[(parent >= 0) & (parent < n)], minlength=n).argmax())
    table[bad] = 5 * n  # a parent with several children whose page is outside the pool
    before, want = pool.clone(), pool.clone()
    lo, to, tk = (torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(3))
    kv.reorder(n, dev(parent), dev(lens), dev(table), 1, dev(spare), lo, to, tk, stream=stream())
    seen = set()
    for r, q in enumerate(parent):
        live = 0 <= q < n
        part = live and lens[q] % page and q in seen and q != bad
        assert lo[r] == (lens[q] if live else 0) and tk[r] == int(bool(part))
        assert to[r] == (-1 if not live or not lens[q] else spare[r] if part else table[q, 0])
        if part:
            want[:, spare[r]] = before[:, table[q, 0]]
        if live:
            seen.add(q)
    assert torch.equal(pool.view(torch.int16), want.view(torch.int16))


def test_reorder_refusals():
    kv, t = e.KvCache(1, 1, 16, 4, 1), torch.zeros(64, device="cuda", dtype=torch.int32)
    ok = dict(n=2, parent=t, length=t[2:], table=t[4:], table_ld=2, spare=t[8:], length_out=t[16:], table_out=t[20:], taken=t[32:])
    kv.reorder(**ok)
    kv.reorder(**(ok | dict(n=0, parent=None)))
    for kw in (dict(n=-1), dict(parent=None), dict(taken=None), dict(table_ld=0), dict(table_ld=-1), dict(table_out=t[4:]), dict(table_out=t[7:]),
               dict(length_out=t[2:]), dict(taken=t)):
        with pytest.raises(ValueError):
            kv.reorder(**(ok | kw))
    with pytest.raises(e.ElbError):
        kv.reorder(**(ok | dict(n=4097)))


# ---------------------------------------------------------------- selection

def select(x, scores, groups, beams, k, allowed=None, v=None, shared=False):
    v = v or x.shape[1]
    d = x.device
    parent, token = (torch.full((groups, k), 77, dtype=torch.int32, device=d) for _ in range(2))
    score = torch.full((groups, k), 77.0, dtype=F64, device=d)
    words = bits = None
    if allowed is not None:
        b = np.packbits(allowed.cpu().numpy(), axis=-1, bitorder="little")
        words = np.zeros((*b.shape[:-1], (v + 31) // 32 * 4), np.uint8)
        words[..., :b.shape[-1]] = b
        bits = torch.from_numpy(words.view(np.int32)).cuda()
    work = torch.full((e.beam_select_work(v, groups, beams, k),), 255, dtype=torch.uint8, device=d)
    e.beam_select(x, v, groups, beams, scores, k, parent, token, score, work, work.numel(), ld=x.stride(0), allowed=bits,
                  allowed_ld=0 if bits is None or shared else bits.shape[-1], stream=stream())
    return parent.cpu().numpy(), token.cpu().numpy(), score.cpu().numpy()


def selected(x, scores, groups, beams, k, allowed=None):
    """The definition: rows sorted by (logit, token), then all rows' candidates by (score, row)."""
    x, scores = x.cpu().numpy().astype(np.float64), scores.cpu().numpy()
    with np.errstate(all="ignore"):
        m = np.max(x, -1, keepdims=True)
        lse = (m + np.log(np.exp(x - m).sum(-1, keepdims=True)))[:, 0]
    out = [np.full((groups, k), -1), np.full((groups, k), -1), np.full((groups, k), -np.inf)]
    for g in range(groups):
        c = []
        for b in range(g * beams, (g + 1) * beams):
            ok = np.flatnonzero((x[b] > -np.inf) & (True if allowed is None else allowed[b if allowed.ndim == 2 else slice(None)].cpu().numpy()))
            for rank, t in enumerate(ok[np.argsort(-x[b, ok], kind="stable")][:k]):
                s = scores[b] + (x[b, t] - lse[b])
                if np.isfinite(s):
                    c.append((-s, b, rank, t))
        for r, (s, b, _, t) in enumerate(sorted(c)[:k]):
            out[0][g, r], out[1][g, r], out[2][g, r] = b, t, -s
    return out


def agree(got, want, n):
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    fine = np.isfinite(want[2])
    assert np.array_equal(got[2][~fine], want[2][~fine])
    # a sum of n exponentials in double (each off by 2^-51, the additions by n 2^-53) and three roundings of the score
    assert (np.abs(got[2][fine] - want[2][fine]) <= (n + 8) * 2.0 ** -52 + 4 * 2.0 ** -52 * np.abs(want[2][fine])).all()


@pytest.mark.parametrize("groups,beams,k,v", [(1, 1, 1, 1), (1, 1, 1, 33), (2, 4, 8, 151936), (3, 5, 10, 4097), (1, 64, 64, 1000), (7, 2, 4, 4096),
                                              (16, 4, 8, 20000), (1, 3, 64, 100), (5, 1, 2, 2), (1, 16, 32, 200001), (2, 33, 3, 77)])
@pytest.mark.parametrize("masked", (False, True))
def test_select(groups, beams, k, v, masked):
    if k > beams * v:
        k = beams * v
    g = gen(28 + v)
    x = randn(g, groups * beams, v) * 4
    scores = torch.randn(groups * beams, generator=g, device="cuda", dtype=F64) * 3 - 20
    allowed = torch.rand(groups * beams, v, generator=g, device="cuda") < 0.5 if masked else None
    agree(select(x, scores, groups, beams, k, allowed), selected(x, scores, groups, beams, k, allowed), v)


def test_select_ties_go_to_the_lowest():
    """Few distinct logits in equal rows: within a row the lower token, between equal scores the lower row."""
    x = torch.randint(0, 3, (4, 9000), generator=gen(29), device="cuda").float()
    x[1], x[3] = x[0], x[2]
    scores = torch.tensor([-1.0, -1.0, -2.0, -2.0], dtype=F64, device="cuda")
    for k in (1, 5, 64):
        agree(select(x, scores, 2, 2, k), selected(x, scores, 2, 2, k), 9000)
    agree(select(x * 0, scores, 2, 2, 64), selected(x * 0, scores, 2, 2, 64), 9000)


def test_select_what_is_no_candidate():
    """-infinity, NaN and +infinity among the logits, beams that do not exist, masks that leave nothing or little."""
    g = gen(30)
    x = randn(g, 6, 5000)
    x[0, ::2] = -math.inf
    x[1] = -math.inf
    x[2, 17] = math.nan
    x[3, 40] = math.inf
    scores = torch.tensor([-5.0, -1.0, -1.0, -1.0, -math.inf, -3.0], dtype=F64, device="cuda")
    agree(select(x, scores, 1, 6, 20), selected(x, scores, 1, 6, 20), 5000)
    allowed = torch.zeros(6, 5000, dtype=torch.bool, device="cuda")
    allowed[0, 4], allowed[0, 7], allowed[5, 4999] = True, True, True  # token 4 of row 0 is -infinity
    got = select(x, scores, 1, 6, 5, allowed)
    agree(got, selected(x, scores, 1, 6, 5, allowed), 5000)
    assert (got[0][0, 2:] == -1).all() and (got[1][0, 2:] == -1).all() and (got[2][0, 2:] == -math.inf).all()
    agree(select(x, scores * math.nan, 1, 6, 5), selected(x, scores * math.nan, 1, 6, 5), 5000)
    one = torch.rand(5000, generator=g, device="cuda") < 0.1
    agree(select(x, scores, 2, 3, 9, one, shared=True), selected(x, scores, 2, 3, 9, one), 5000)


@pytest.mark.parametrize("size", (1e-3, 80.0, 1e30))
def test_select_sizes_and_strides(size):
    """Flat, steep and huge logits, in rows that are further apart than their length and start anywhere."""
    buf = randn(gen(31), 6 * 7003 + 1) * size
    x = buf[1:].view(6, 7003)[:, :6999]
    scores = torch.linspace(-3, 0, 6, dtype=F64, device="cuda")
    agree(select(x, scores, 2, 3, 6, v=6999), selected(x, scores, 2, 3, 6), 6999)


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("kind", (e.KV_F16, e.KV_PAIR))
def test_a_beam_search_over_the_pages(kind):
    """Prompts, then steps of append, attention, selection and reordering: every beam's output is
    that of its own history of keys and values, kept in 64 bits beside it."""
    groups, beams, hkv, h, page, steps, v = 2, 3, 2, 4, 16, 20, 500
    rows, prompt = groups * beams, (13, 30)
    g = gen(32)
    rope = e.Rope(D)
    pages = 400
    pool = torch.zeros((1, pages, 2, hkv, kind, page, D), dtype=torch.half, device="cuda")
    kv = e.KvCache(1, hkv, page, pages, kind, mem=pool)
    free = list(range(pages))[::-1]
    width = 8
    table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    length = torch.zeros(rows, dtype=torch.int32, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    head = randn(g, h * D, v) * 0.2
    stored = lambda: pool[0]

    def history(r):
        n = int(length[r])
        pg = table[r, :(n + page - 1) // page].long()
        return stored()[pg].to(F64).sum(3).permute(1, 2, 0, 3, 4).reshape(2, hkv, -1, D)[:, :, :n]

    def step(n_seq, nq, lens, tab, x):
        n = x.shape[0]
        b = e.KvBatch(n_seq, n, max(nq), max(lens), i32(np.concatenate([[0], np.cumsum(nq)]).tolist()), i32(lens), tab, width)
        q, out = torch.empty(n, h * D, device="cuda"), torch.empty(n, h * D, device="cuda")
        a, ld = x.data_ptr(), x.shape[1]
        kv.append(0, b, a + 4 * h * D, a + 4 * (h + hkv) * D, ld, ld, rope=rope, q=a, ldq=ld, n_head=h, q_out=q, ldqo=h * D, stream=stream())
        work = torch.empty(kv.attention_work(b, h), dtype=torch.uint8, device="cuda")
        kv.attention(0, b, q, out, h, 1 / math.sqrt(D), work, work.numel(), stream=stream())
        return q, out

    for s, n in enumerate(prompt):  # prompts into the first beam of each group
        for i in range((n + page - 1) // page):
            table[s * beams, i] = free.pop()
    first = [0, beams]
    x = randn(g, sum(prompt), (h + 2 * hkv) * D)
    step(2, prompt, prompt, table[first].contiguous(), x)
    length[first] = i32(list(prompt))
    kept = {r: history(r).clone() for r in first}
    scores = torch.full((rows,), -math.inf, dtype=F64, device="cuda")
    scores[first] = 0
    parent = i32([r // beams * beams for r in range(rows)])  # every beam from its group's prompt
    for t in range(steps):
        spare = i32([free.pop() for _ in range(rows)])
        lo, to, tk = torch.empty_like(length), torch.empty_like(table), torch.empty_like(length)
        kv.reorder(rows, parent, length, table, width, spare, lo, to, tk, stream=stream())
        length, table = lo, to
        kept = {r: kept[int(parent[r])].clone() for r in range(rows) if int(parent[r]) in kept}
        for r in range(rows):
            if int(length[r]) % page == 0:
                table[r, int(length[r]) // page] = free.pop()
        length = length + 1
        x = randn(g, rows, (h + 2 * hkv) * D)
        q, out = step(rows, [1] * rows, length.tolist(), table, x)
        for r in range(rows):
            mine = history(r)
            assert torch.equal(mine[:, :, :-1], kept[r])  # its own past, whoever else goes on from there
            kept[r] = mine.clone()
            for i in range(h):
                k, val = mine[:, i // (h // hkv)]
                qi = q[r, i * D:(i + 1) * D].to(F64)
                w = (k @ qi / math.sqrt(D)).softmax(0)
                d = float((k.abs() @ qi.abs()).max() / math.sqrt(D)) * 28 * 2.0 ** -23
                assert ((out[r, i * D:(i + 1) * D].to(F64) - w @ val).abs() <= (w @ val.abs()) * (2 * d + 100 * U)).all()
        logits = out @ head
        p, tok, sc = select(logits, scores, groups, beams, beams)
        if t == 0:
            assert (p == [[0] * beams, [beams] * beams]).all()  # only the first beams live so far
        scores = torch.from_numpy(sc.reshape(-1)).cuda()
        parent = i32(p.reshape(-1).tolist())
