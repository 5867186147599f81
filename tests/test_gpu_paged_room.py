"""A paged model that lacks pages or device memory: the call is refused and leaves every sequence as it was. Its decode loop."""
import ctypes as C

import numpy as np
import pytest

import exactinfer_b200 as e
import test_gpu_paged_model as base
from exactinfer_b200 import capi, synth

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def models():
    spec = base.spec_of("q4_k_m")
    tens = list(synth.generate(spec, 17))
    make = lambda n_ctx=96, **kw: e.Backend(spec, tens, n_ctx, max_batch=32, n_seq=6, **kw)
    return spec, make, make()


@pytest.mark.parametrize("pos0", (0, 7, 20))
@pytest.mark.parametrize("call", ("eval", "eval_top", "eval_steps"))
def test_a_prompt_of_several_chunks_that_runs_out_of_pages(models, call, pos0):
    """Pages for the first chunk, not for all: nothing is evaluated, and the sequence is as long as before."""
    spec, make, flat = models
    rng = np.random.default_rng(30)
    paged = make(pages=(16, 4, e.KV_PAIR))
    toks = rng.integers(0, spec.n_vocab, 96)
    for model in (paged, flat):
        base.prompt(model, 0, toks[:20])
        base.prompt(model, 1, toks[:16])
    more = rng.integers(0, spec.n_vocab, 60)
    with pytest.raises(MemoryError):
        {"eval": lambda: paged.eval(more, pos0), "eval_top": lambda: paged.eval_top(more, pos0, 3), "eval_steps": lambda: paged.eval_steps(more, pos0)}[call]()
    assert paged.free_pages() == 1
    assert base.rel(paged.eval(toks[20:22], 20), flat.eval(toks[20:22], 20)) <= base.REL_TOL
    # what does fit: all four pages but the other sequence's
    assert base.rel(paged.eval(more[:48], 0), flat.eval(more[:48], 0)) <= base.REL_TOL


@pytest.fixture
def full_device():
    """Calls that take all free device memory, down to pieces of 512 bytes, and give it back."""
    held = []

    def fill():
        for size in (1 << 30, 1 << 26, 1 << 21, 1 << 16, 1 << 12, 512):
            while True:
                p = C.c_void_p()
                if capi.lib().elb_malloc(0, size, C.byref(p)):
                    break
                held.append(p)

    def give_back():
        while held:
            capi.lib().elb_free(held.pop())

    yield fill, give_back
    give_back()


@pytest.mark.parametrize("call", ("eval", "eval_batch"))
def test_no_device_memory_for_working_space(models, full_device, call):
    """Longer contexts need more of it: without any the call is refused before a length or a table changes, and succeeds later."""
    spec, make, _ = models
    fill, give_back = full_device
    flat, paged = make(n_ctx=1200), make(n_ctx=1200, pages=(16, 160, e.KV_PAIR))
    rng = np.random.default_rng(31)
    toks = rng.integers(0, spec.n_vocab, 1100)
    paged.eval(toks[:505], 0)
    free = paged.free_pages()
    fill()
    with pytest.raises(MemoryError):
        if call == "eval":
            paged.eval(toks[200:1100], 200)
        else:
            rows = np.concatenate([toks[:16], toks[500:515]])
            paged.eval_batch(rows, [1] * 16 + [0] * 15, list(range(16)) + list(range(500, 515)), [0] * 30 + [1])
    assert paged.free_pages() == free
    give_back()
    want = flat.eval(toks, 0)
    assert base.rel(paged.eval(toks[505:], 505), want) <= base.REL_TOL


def test_a_shared_last_page_is_copied_without_an_allocation(models, full_device):
    spec, make, flat = models
    fill, give_back = full_device
    paged = make(pages=(16, 20, e.KV_PAIR))
    rng = np.random.default_rng(32)
    toks = rng.integers(0, spec.n_vocab, 40)
    for s in (0, 1):
        base.prompt(flat, s, toks[:32])
    base.prompt(paged, 0, toks[:32])
    paged.reorder([1], [0])
    want = flat.eval_batch(toks[32:40], [0] * 4 + [1] * 4, list(range(20, 24)) * 2, [0, 0, 0, 1] * 2)
    paged.eval_batch(toks[:1], [3], [0])  # (every kernel of the call has run)
    fill()
    got = paged.eval_batch(toks[32:40], [0] * 4 + [1] * 4, list(range(20, 24)) * 2, [0, 0, 0, 1] * 2)
    give_back()
    assert base.rel(got, want) <= base.REL_TOL


def test_beams_that_fill_the_pool_go_on_from_one_of_them(models):
    """No page is free, but the call itself gives up three half-filled ones: they take the copies."""
    spec, make, flat = models
    rng = np.random.default_rng(33)
    paged = make(pages=(16, 5, e.KV_PAIR))
    toks, own = rng.integers(0, spec.n_vocab, 16), rng.integers(0, spec.n_vocab, (5, 4))
    base.prompt(paged, 0, toks)
    paged.reorder([1, 2, 3], [0, 0, 0])
    for i in range(5):
        paged.eval_batch(own[i], range(4), [16 + i] * 4)
    assert paged.free_pages() == 0
    paged.reorder(range(4), [2, 2, 2, 2])
    assert paged.free_pages() == 0
    for s in range(4):
        base.prompt(flat, s, np.concatenate([toks, own[:, 2]]))
    for step in range(4):
        nxt = rng.integers(0, spec.n_vocab, 4)
        a, b = paged.eval_batch(nxt, range(4), [21 + step] * 4), flat.eval_batch(nxt, range(4), [21 + step] * 4)
        assert base.rel(a, b) <= base.REL_TOL
    with pytest.raises(MemoryError):
        paged.reorder([4], [0])  # this one needs a page more than there are


def test_steps_form_their_logits(models):
    """eval_steps is a decode loop without reading back: every step is all of a step, the output head as well."""
    spec, make, flat = models
    rng = np.random.default_rng(34)
    toks = rng.integers(0, spec.n_vocab, 12)
    for model in (make(pages=(16, 8, e.KV_PAIR)), flat):
        model.eval(toks[:5], 0)
        model.eval(toks[5:6], 5)
        one = model.last_eval_stats()[1]
        model.eval_steps(toks[6:9], 6)
        ms, launches = model.last_eval_stats()
        assert launches == 3 * one and ms > 0
