"""Sessions with drafted trees where the calls around them matter: page pools that run out, threads."""
from concurrent.futures import ThreadPoolExecutor

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


def test_sessions_that_share_pages_on_two_threads(cuda_ok):
    """Two sessions forked from one prompt write their first positions, trees and steps, on threads of their own:
    the copy of the page they share is done before the other one writes it."""
    cfg = spmodel.CONFIGS["micro_gemma"]
    m = spb200.Model.upload(cfg, spmodel.gen_model(cfg, seed=5))
    pool = spb200.KvPool(m, 128, 8)
    prompt = spmodel.gen_tokens(62, 100, cfg.n_vocab)

    def go(h, first):
        res = h.tree_step([first, first + 1, first + 2], [-1, 0, 0])
        rows = [res.logits.copy()]
        h.tree_commit([0, 2])
        rows += [h.step(first + 3 + i).copy()[None] for i in range(3)]
        return np.concatenate(rows)

    def fork():
        a = pool.session(300)
        a.prefill(prompt, logits=False)
        return a, a.clone()

    a, b = fork()
    want = [go(a, 5), go(b, 50)]
    a.close()
    b.close()
    with ThreadPoolExecutor(2) as ex:
        for _ in range(40):
            hs = fork()
            got = list(ex.map(go, hs, (5, 50)))
            for g, w, h in zip(got, want, hs):
                assert np.array_equal(u32(g), u32(w))
                h.close()
    assert pool.free_pages() == 8
    pool.free()
    m.free()
