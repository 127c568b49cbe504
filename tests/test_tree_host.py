"""Refusals of the tree-verification entry points that need no GPU."""
import ctypes as C

import numpy as np
import pytest

import spb200


def view(**kw):
    a = np.zeros(64, np.int32)
    d = dict(k=256, v=256, ptab=256, n_pages=4, page=16, ptab_ld=2, n_layers=1, n_head_kv=2, head_dim=64) | kw
    v = spb200.KvView(*d.values())
    v._keep = a
    return v


def rc(f, *a):
    try:
        f(*a)
        return 0
    except spb200.SpbError as e:
        return e.code


BAD, UNS = spb200.SPB_EBADARG, spb200.SPB_EUNSUPPORTED


@pytest.mark.parametrize("kw,code", [
    (dict(k=None), BAD), (dict(v=None), BAD), (dict(n_pages=0), BAD), (dict(page=0), BAD), (dict(page=-8), BAD), (dict(ptab_ld=0), BAD),
    (dict(n_layers=0), BAD), (dict(n_head_kv=0), BAD), (dict(head_dim=96), UNS), (dict(head_dim=32), UNS),
    (dict(k=260), BAD), (dict(v=272), BAD), (dict(ptab=None, n_pages=1), BAD),
])
def test_cache_views_are_checked(kw, code):
    v = view(**kw)
    assert rc(spb200.tree_attn, v, 0, 2, 256, 256, 256, 2, 8, 256, 4, -1, 256) == code
    assert rc(spb200.kv_compact, v, 2, 256, 256, 256, 2) == code


@pytest.mark.parametrize("args,code", [
    (dict(layer=1), BAD), (dict(layer=-1), BAD), (dict(n_seq=-1), BAD), (dict(rows=-1), BAD), (dict(rows=129), BAD), (dict(max_ctx=-1), BAD),
    (dict(n_head=3), UNS), (dict(n_head=18), UNS), (dict(n_head=0), UNS), (dict(ctx=None), BAD), (dict(row0=None), BAD),
    (dict(parent=None), BAD), (dict(q=None), BAD), (dict(out=None), BAD), (dict(q=260), BAD),
])
def test_attention_refusals(monkeypatch, args, code):
    d = dict(layer=0, n_seq=2, ctx=256, row0=256, parent=256, rows=2, max_ctx=8, q=256, n_head=4, window=-1, out=256) | args
    assert rc(spb200.tree_attn, view(), *d.values()) == code


def test_host_memory_is_refused():
    """Pointers that are no device memory come back as an error, not as a fault (256 is no allocation at all)."""
    a = np.zeros(4096, np.int32)
    p = (a.ctypes.data + 15) & ~15
    v = view(k=p, v=p, ptab=p)
    assert rc(spb200.tree_attn, v, 0, 2, p, p, p, 2, 8, p, 4, -1, p) == BAD
    assert rc(spb200.kv_compact, v, 2, p, p, p, 2) == BAD
    assert rc(spb200.logprobs, p, 1, 8, 8, p, p, 1, p, p, p, 0, None, None) == BAD


@pytest.mark.parametrize("args", [
    dict(rows=-1), dict(vocab=0), dict(ld=7), dict(n_tok=-1), dict(top=-1), dict(top=33), dict(logits=None), dict(tok=None),
    dict(logprob=None), dict(top=2, top_id=None), dict(top=2, top_logprob=None), dict(rows=0), dict(tok_row=None, n_tok=5),
])
def test_logprob_refusals(args):
    d = dict(logits=256, rows=4, vocab=8, ld=8, tok_row=256, tok=256, n_tok=2, logprob=256, lse=256, entropy=256, top=0, top_id=256,
             top_logprob=256) | args
    assert rc(spb200.logprobs, *d.values()) == BAD


@pytest.mark.parametrize("max_ctx,window,code", [(1048513, -1, UNS), (1 << 29, 1048513, UNS), ((1 << 30) + 1, 1024, UNS),
                                                 ((1 << 31) - 1, 64, UNS), (1 << 30, 1024, BAD)])   # (the last: only its pointers are bad)
def test_attention_limits(max_ctx, window, code):
    assert rc(spb200.tree_attn, view(), 0, 2, 256, 256, 256, 2, max_ctx, 256, 4, window, 256) == code


@pytest.mark.parametrize("args", [dict(vocab=(1 << 22) + 1, ld=1 << 23), dict(rows=(1 << 26) + 1), dict(n_tok=(1 << 26) + 1),
                                  dict(n_tok=(1 << 31) - 1)])
def test_logprob_limits(args):
    d = dict(logits=256, rows=4, vocab=8, ld=8, tok_row=256, tok=256, n_tok=2, logprob=256, lse=256, entropy=256, top=0, top_id=256,
             top_logprob=256) | args
    assert rc(spb200.logprobs, *d.values()) == UNS


def test_nothing_to_do():
    assert rc(spb200.logprobs, None, 0, 8, 8, None, None, 0, None, None, None, 0, None, None) == 0


def test_session_calls_refuse_null():
    L = spb200.load()
    n = np.array([1], np.int32)
    out = spb200.StepOut()
    assert L.spb_batch_tree_step(None, 1, n.ctypes.data, n.ctypes.data, n.ctypes.data, None) == BAD
    hs = (C.c_void_p * 1)(None)
    for B in (0, -1, 65):
        assert L.spb_batch_tree_step(hs, B, n.ctypes.data, n.ctypes.data, n.ctypes.data, C.byref(out)) == BAD
    assert L.spb_batch_tree_step(hs, 1, n.ctypes.data, n.ctypes.data, n.ctypes.data, C.byref(out)) == BAD
    assert L.spb_session_tree_commit(None, n.ctypes.data, 1) == BAD
    assert L.spb_session_score(None, n.ctypes.data, 1, C.byref(out)) == BAD


def test_step_results_are_split_by_session():
    r = spb200.StepResult(5, 7, 2, logits=True)
    a = r.rows(1, 3)
    assert a.logits.shape == (2, 7) and a.top_id.shape == (2, 2) and a.entropy.base is r.entropy
    with pytest.raises(ValueError):
        spb200.batch_tree_step([type("S", (), {"h": None, "V": 8})()], [[1, 2]], [[-1]])
