"""A paged model that lacks pages or device memory: the call is refused and leaves every sequence as it was."""
import numpy as np
import pytest

import exactinfer_b200 as e
import test_gpu_paged_model as base
from exactinfer_b200 import synth

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
