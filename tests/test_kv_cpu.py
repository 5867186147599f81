"""Rotary frequencies, sizes and refusals of the paged-cache calls that need no GPU."""
import ctypes as C
import math

import numpy as np
import pytest

import exactinfer_b200 as e
from exactinfer_b200 import capi


@pytest.fixture(scope="module", autouse=True)
def lib():
    from exactinfer_b200 import build
    build.build()
    return capi.lib()


def formula(c):
    """The scaled frequencies from their definition, pair by pair."""
    out = []
    for i in range(c.dim // 2):
        f = c.base ** (-2.0 * i / c.dim)
        if c.scaling == e.ROPE_LINEAR:
            f /= c.factor
        if c.scaling == e.ROPE_YARN:
            at = lambda b: c.dim / 2 * math.log(c.orig_ctx / (b * 2 * math.pi), c.base)
            lo, hi = max(math.floor(at(c.beta_fast)), 0), min(math.ceil(at(c.beta_slow)), c.dim - 1)
            r = min(1.0, max(0.0, (i - lo) / (hi - lo if hi != lo else 0.001)))
            f = r * f / c.factor + (1 - r) * f
        if c.scaling == e.ROPE_BANDS:
            wave = 2 * math.pi / f
            if wave > c.orig_ctx / c.low_freq:
                f /= c.factor
            elif wave >= c.orig_ctx / c.high_freq:
                s = (c.orig_ctx / wave - c.low_freq) / (c.high_freq - c.low_freq)
                f = (1 - s) * f / c.factor + s * f
        out.append(f)
    return np.array(out)


@pytest.mark.parametrize("dim", (2, 6, 64, 128))
@pytest.mark.parametrize("scaling", (e.ROPE_PLAIN, e.ROPE_LINEAR, e.ROPE_YARN, e.ROPE_BANDS))
def test_frequencies(dim, scaling):
    c = e.rope_config(128, dim=dim, base=1e6, scaling=scaling, factor=4.0, orig_ctx=32768.0)
    f, m = e.rope_frequencies(c)
    # pow, log and a few products in double on both sides: each off by a few units of 2^-53, the exponent's error times ln(base)
    assert np.allclose(f, formula(c), rtol=64 * 2**-53, atol=0)
    want = 0.1 * math.log(4.0) + 1.0 if scaling == e.ROPE_YARN else 1.0
    assert abs(m - want) <= 4 * 2**-53
    if scaling == e.ROPE_YARN:
        assert e.rope_frequencies(e.rope_config(128, scaling=scaling, factor=4.0, orig_ctx=32768.0, attn_factor=1.5))[1] == 1.5


def test_frequencies_ends_meet():
    """YaRN and the bands keep fast pairs and divide slow ones; a factor of 1 changes nothing."""
    plain, _ = e.rope_frequencies(e.rope_config())
    for scaling in (e.ROPE_YARN, e.ROPE_BANDS):
        f, _ = e.rope_frequencies(e.rope_config(scaling=scaling, factor=4.0, orig_ctx=32768.0))
        assert f[0] == plain[0] and f[-1] == plain[-1] / 4.0
        f, _ = e.rope_frequencies(e.rope_config(scaling=scaling, factor=1.0, orig_ctx=32768.0))
        assert np.allclose(f, plain, rtol=4 * 2**-53, atol=0)


@pytest.mark.parametrize("bad", (dict(head_dim=0), dict(head_dim=258), dict(head_dim=127), dict(dim=130), dict(dim=3), dict(dim=0), dict(layout=2),
                                 dict(scaling=4), dict(base=1.0), dict(base=float("nan")), dict(scaling=1, factor=0.5),
                                 dict(scaling=2, factor=4.0), dict(scaling=2, factor=4.0, orig_ctx=1e4, beta_slow=0.0),
                                 dict(scaling=2, factor=4.0, orig_ctx=1e4, attn_factor=-1.0),
                                 dict(scaling=3, factor=4.0, orig_ctx=1e4, low_freq=4.0), dict(scaling=1, factor=float("inf"))))
def test_rope_refuses(lib, bad):
    c = e.rope_config(**bad)
    h = C.c_void_p()
    assert lib.elb_rope_create(0, C.byref(c), C.byref(h)) == capi.ERR_INVALID and not h
    with pytest.raises(ValueError):
        e.rope_frequencies(c)


def test_pool_sizes():
    assert e.KvCache.bytes(36, 8, 16, 100, e.KV_F16) == 36 * 100 * 2 * 8 * 16 * 128 * 2
    assert e.KvCache.bytes(36, 8, 64, 100, e.KV_PAIR) == 36 * 100 * 2 * 8 * 2 * 64 * 128 * 2
    for args in ((0, 8, 16, 1, 1), (1, 0, 16, 1, 1), (1, 8, 24, 1, 1), (1, 8, 512, 1, 1), (1, 8, 16, 0, 1), (1, 8, 16, 1, 3), (64, 64, 256, 4096, 2)):
        assert e.KvCache.bytes(*args) == 0
    assert e.KvCache.bytes(1, 8, 16, 1, 1, head_dim=64) == 0


@pytest.mark.parametrize("args,code", (((0, 1, 2, 64, 16, 4, 1, None), capi.ERR_UNSUPPORTED), ((0, 1, 2, 128, 48, 4, 1, None), capi.ERR_UNSUPPORTED),
                                       ((0, 1, 2, 128, 16, 4, 0, None), capi.ERR_UNSUPPORTED), ((0, 0, 2, 128, 16, 4, 1, None), capi.ERR_INVALID),
                                       ((0, 1, 2, 128, 16, -4, 1, None), capi.ERR_INVALID), ((0, 64, 64, 128, 256, 4096, 2, None), capi.ERR_UNSUPPORTED),
                                       ((0, 1, 2, 128, 16, 4, 1, 4096 + 64), capi.ERR_INVALID)))
def test_cache_refuses(lib, args, code):
    h = C.c_void_p()
    assert lib.elb_kv_create(*args, C.byref(h)) == code and not h
    assert lib.elb_last_error()
    assert lib.elb_kv_create(*args, None) == capi.ERR_INVALID


def test_null_handles_are_refused(lib):
    b = e.KvBatch(1, 1, 1, 1, 256, 256, 256, 1)
    assert lib.elb_kv_attention_work(None, b._as_parameter_, 8) == 0
    assert lib.elb_kv_attention_dev(None, 0, b._as_parameter_, None, 0, 8, 1.0, None, 0, None, 0, None) == capi.ERR_INVALID
    assert lib.elb_kv_append_dev(None, 0, b._as_parameter_, None, None, 0, None, 0, None, 0.0, None, 0, 0, None, None, 0, None) == capi.ERR_INVALID
    assert lib.elb_kv_reorder_dev(None, 1, None, None, None, 1, None, None, None, None, None) == capi.ERR_INVALID
    assert lib.elb_rope_dev(None, None, 0, None, 0, 1, 1, None, None, 0.0, None) == capi.ERR_INVALID
    assert lib.elb_kv_memory(None) is None
    lib.elb_kv_destroy(None)
    lib.elb_rope_destroy(None)


def test_beam_select_refuses(lib):
    assert e.beam_select_work(1000, 2, 4, 8) >= 256
    for bad in ((0, 1, 4, 8), (1000, -1, 4, 8), (1000, 1, 0, 8), (1000, 1, 65, 8), (1000, 1, 4, 0), (1000, 1, 4, 65), (1000, 2000, 64, 4)):
        assert e.beam_select_work(*bad) == 0
    p, w = 4096, e.beam_select_work(1000, 2, 4, 8)
    call = lambda ld=1000, v=1000, g=2, b=4, sc=p, al=None, ald=0, k=8, out=p, work=p, wb=w: lib.elb_beam_select_dev(
        0, p, ld, v, g, b, sc, al, ald, k, out, out, out, work, wb, None)
    for kw, code in ((dict(ld=999), capi.ERR_INVALID), (dict(k=0), capi.ERR_INVALID), (dict(k=65), capi.ERR_INVALID), (dict(v=1, ld=1, k=5), capi.ERR_INVALID),
                     (dict(b=65), capi.ERR_INVALID), (dict(sc=None), capi.ERR_INVALID), (dict(out=None), capi.ERR_INVALID),
                     (dict(work=None), capi.ERR_INVALID), (dict(wb=w - 1), capi.ERR_INVALID), (dict(work=p + 8), capi.ERR_INVALID),
                     (dict(al=p, ald=31), capi.ERR_INVALID), (dict(g=70000, b=1, k=1), capi.ERR_UNSUPPORTED), (dict(g=0), capi.OK)):
        assert call(**kw) == code, kw
    ok, _ = e.cuda_available()
    if not ok:
        assert call() == capi.ERR_CUDA
