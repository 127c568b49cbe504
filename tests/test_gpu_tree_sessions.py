"""Sessions with drafted trees where the calls around them matter: page pools that run out."""
import numpy as np
import pytest

import spb200
import spmodel
import xref
from test_gpu_tree import u32

pytestmark = pytest.mark.gpu


def test_a_step_without_room_changes_nothing(xr, cuda_ok):
    """A pool with one free page, a write that needs two (a copy of the shared page and a new one): the call
    fails, takes no page, and the sessions that share the page go on apart from each other."""
    cfg = spmodel.CONFIGS["micro_gemma"]
    T = spmodel.gen_model(cfg, seed=5)
    m = spb200.Model.upload(cfg, T)
    pool = spb200.KvPool(m, 128, 3)
    prompt, other = spmodel.gen_tokens(62, 120, cfg.n_vocab), spmodel.gen_tokens(63, 10, cfg.n_vocab)
    s, t = pool.session(400), pool.session(100)
    t.prefill(other, logits=False)
    s.prefill(prompt, logits=False)
    c = s.clone()
    assert pool.free_pages() == 1
    for call in (lambda: s.tree_step([3] * 20, [-1] * 20), lambda: s.score([3] * 20), lambda: s.prefill([3] * 20), lambda: s.greedy(3, 20),
                 lambda: spb200.batch_tree_step([t, s], [[1], [3] * 20], [[-1], [-1] * 20])):
        with pytest.raises(spb200.SpbError) as e:
            call()
        assert e.value.code == spb200.SPB_EOOM and pool.free_pages() == 1 and s.position() == 120
    xs = xr.session(xref.build_desc(cfg, T), 400)
    xs.prefill(prompt, all_logits=False)
    xc, xt = xs.clone(), xr.session(xref.build_desc(cfg, T), 400)
    xt.prefill(other, all_logits=False)
    for i in range(4):                                       # s copies the page at its first token, c writes the old one
        for h, x, tok in ((s, xs, 10 + i), (c, xc, 20 + i), (t, xt, 30 + i)):
            assert np.array_equal(u32(h.step(tok)), u32(x.step(tok))), i
    for h in (s, c, t, xs, xc, xt):
        h.close()
    assert pool.free_pages() == 3
    pool.free()
    m.free()
