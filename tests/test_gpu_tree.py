"""Verifying drafted trees on the GPU: attention of a tree's nodes over a cache, log probabilities
with entropy and alternatives, the move of an accepted path's rows, and the three as one step.

The attention's oracle is the written contract in whole numbers (numpy int64 and Python integers),
the sessions' is XREF decoding every path token by token: both byte for byte. Log probabilities are
compared with 64-bit floating point; their tolerance counts roundings (see `lp_tol`)."""
import ctypes as C

import numpy as np
import pytest
import torch

import spb200
import spmodel
import xref

pytestmark = pytest.mark.gpu

ONE = 1 << 30
EXP2 = [1073741824, 744261118, 257941248, 59597083, 10327387, 1431680, 165394]


def u32(a):
    return np.ascontiguousarray(a).view(np.uint32)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def errs():
    return spb200.load().spb_take_device_errors()


# ------------------------------------------------------------------------------ the contract
def exp_fixed(far):
    """e of `far` >= 0 grid steps (2^-14) below the maximum, in 2^30 fixed point."""
    far = np.minimum(far, 1 << 19)
    g = (far * 1549082005 + 16383) >> 14
    n, r = g >> 30, g & (ONE - 1)
    acc = np.full_like(r, EXP2[6])
    for k in range(5, -1, -1):
        acc = ((acc * (ONE - r)) >> 30) + EXP2[k]
    n2 = np.minimum(n, 40)
    return np.where(n >= 32, 0, np.where(r > 0, acc >> (n2 + 1), ONE >> n2))


def chain(parent, i):
    c = [i]
    while parent[c[-1]] >= 0:
        c.append(parent[c[-1]])
    return c[::-1]


def attend(K, V, q, ctx, parent, win, G):
    """K, V [slots][NKV][HD], q [n][NKV*G*HD] int: out [n][NKV*G*HD] f32."""
    n, NKV, HD = len(parent), K.shape[1], K.shape[2]
    asc = np.float32(1.0) / np.sqrt(np.float32(HD))
    out = np.zeros((n, NKV, G, HD), np.float32)
    for i in range(n):
        c = chain(parent, i)
        first = max(0, ctx + len(c) - 1 - win + 1) if win > 0 else 0
        see = list(range(min(first, ctx), ctx)) + [ctx + a for t, a in enumerate(c) if ctx + t >= first]
        for g in range(NKV):
            k, v = K[see, g].astype(np.int64), V[see, g].astype(object)
            for h in range(G):
                qq = q[i].reshape(NKV, G, HD)[g, h].astype(np.int64)
                s = (k * qq).sum(1)
                z = (s.astype(np.float64) * 2.0 ** -32).astype(np.float32) * asc
                z = z.astype(np.float64) * 16384.0
                zi = np.where(z < 0, np.ceil(z - 0.5), np.floor(z + 0.5)).astype(np.int64)
                e = exp_fixed(zi.max() - zi)
                S = int(e.sum())
                N = (e.astype(object)[:, None] * v).sum(0)
                out[i, g, h] = [np.float32(float((int(x) << 16) // S) * 2.0 ** -32) for x in N]
    return out.reshape(n, NKV * G * HD)


def tree(r, n, chainy=0.0):
    return [-1 if i == 0 or r.random() < 0.15 else int(i - 1 if r.random() < chainy else r.integers(0, i)) for i in range(n)]


class Case:
    """A pool of pages with the given sequences in it (contexts and parents), and their queries."""

    def __init__(self, seed, NKV, G, HD, page, ctx, trees, layers=1, layer=0, scale=1.5, spare=2):
        r = self.r = np.random.default_rng(seed)
        self.NKV, self.G, self.HD, self.page, self.layer, self.ctx, self.trees = NKV, G, HD, page, layer, ctx, trees
        per = [max(1, -(-(c + len(t)) // page)) for c, t in zip(ctx, trees)]
        n_pages, self.ld = sum(per) + spare, max(per)
        order = r.permutation(n_pages)
        self.tab = np.zeros((len(ctx), self.ld), np.int32)
        at = 0
        for b, p in enumerate(per):
            self.tab[b, :p] = order[at:at + p]
            at += p
        lim = (1 << 24) - 1
        shape = (n_pages, layers, NKV, page, HD)
        self.k = np.clip(np.rint(r.standard_normal(shape) * 65536), -lim, lim).astype(np.int32)
        self.v = np.clip(np.rint(r.standard_normal(shape) * 65536 * 3), -lim, lim).astype(np.int32)
        self.rows = sum(len(t) for t in trees)
        self.q = np.clip(np.rint(r.standard_normal((self.rows, NKV * G * HD)) * 65536 * scale), -lim, lim).astype(np.int32)
        self.row0 = np.cumsum([0] + [len(t) for t in trees]).astype(np.int32)
        self.parent = np.array(sum(trees, []), np.int32)

    def upload(self):
        self.d = {n: dev(getattr(self, n)) for n in ("k", "v", "tab", "q", "row0", "parent")}
        self.d["ctx"] = dev(np.array(self.ctx, np.int32))
        self.view = spb200.KvView(self.d["k"].data_ptr(), self.d["v"].data_ptr(), self.d["tab"].data_ptr(), self.k.shape[0],
                                  self.page, self.ld, self.k.shape[1], self.NKV, self.HD)
        return self

    def run(self, win=-1, out=None, stream=None, max_ctx=None):
        d = self.d
        if out is None:
            out = torch.full((self.rows, self.NKV * self.G * self.HD), 7.0, device="cuda")
        spb200.tree_attn(self.view, self.layer, len(self.ctx), d["ctx"].data_ptr(), d["row0"].data_ptr(), d["parent"].data_ptr(),
                         self.rows, max(self.ctx) if max_ctx is None else max_ctx, d["q"].data_ptr(), self.NKV * self.G, win,
                         out.data_ptr(), stream)
        return out

    def want(self, win=-1):
        res = []
        for b, c in enumerate(self.ctx):
            slots = np.arange(c + len(self.trees[b]))
            pg, off = self.tab[b, slots // self.page], slots % self.page
            K, V = self.k[pg, self.layer, :, off], self.v[pg, self.layer, :, off]
            res.append(attend(K, V, self.q[self.row0[b]:self.row0[b + 1]], c, self.trees[b], win, self.G))
        return np.concatenate(res)


@pytest.mark.parametrize("NKV,G,HD,page,ctx,nodes,win", [
    (1, 1, 64, 128, [0], [1], -1),                    # one token, no context
    (2, 4, 64, 24, [37], [13], -1),                   # pages that end inside every tile
    (1, 2, 256, 128, [1], [3], -1),
    (2, 2, 256, 7, [100], [17], -1),                  # a page shorter than a matrix tile
    (1, 8, 128, 128, [129], [9], -1),
    (1, 3, 64, 50, [70], [11], -1),                   # three query heads to a KV head
    (2, 4, 128, 64, [300], [33], -1),
    (1, 4, 64, 4096, [200], [64], -1),                # the largest tree
    (1, 2, 64, 32, [90], [20], 16),                   # window inside the context
    (1, 2, 64, 32, [90], [40], 3),                    # window shorter than the tree is deep
    (1, 2, 64, 32, [5], [12], 1),                     # every node sees itself alone
    (1, 2, 128, 16, [0, 130, 3, 64], [5, 0, 1, 30], -1),   # ragged sequences, one without nodes, one without context
    (2, 2, 64, 48, [17, 200, 48], [8, 8, 8], 20),
])
def test_attention_is_the_contract(cuda_ok, NKV, G, HD, page, ctx, nodes, win):
    errs()
    r = np.random.default_rng(7)
    chainy = 1.0 if win == 3 else 0.5
    c = Case(11, NKV, G, HD, page, ctx, [tree(r, n, chainy) for n in nodes], layers=3, layer=1).upload()
    got = c.run(win).cpu().numpy()
    assert errs() == 0
    assert np.array_equal(u32(got), u32(c.want(win)))


@pytest.mark.parametrize("HD,G,ctx,nodes", [(64, 2, 1500, 6), (256, 2, 700, 20), (128, 4, 2600, 3), (64, 2, 18000, 3), (256, 1, 17500, 2)])
def test_attention_long_contexts(cuda_ok, HD, G, ctx, nodes):
    c = Case(3, 1, G, HD, 128, [ctx], [tree(np.random.default_rng(1), nodes, 0.7)]).upload()
    assert np.array_equal(u32(c.run().cpu().numpy()), u32(c.want()))


def test_attention_extreme_values(cuda_ok):
    """Grid values at the contract's limits (scores stay inside |z| < 2^17), a far outlier, equal scores."""
    errs()
    c = Case(5, 1, 2, 64, 32, [150], [tree(np.random.default_rng(2), 21)])
    lim = (1 << 24) - 1
    c.k[...] = np.where(c.r.random(c.k.shape) < 0.5, lim, -lim)
    c.v[...] = np.where(c.r.random(c.v.shape) < 0.5, (1 << 30) - 1, -(1 << 30) + 1)
    c.q[...] = np.where(c.r.random(c.q.shape) < 0.5, 1, -1) * c.r.integers(0, 200, c.q.shape)
    c.q[0] = lim // 64                      # one large query
    c.q[1] = 0                              # all scores equal: every e is 2^30
    c.upload()
    got = c.run().cpu().numpy()
    assert errs() == 0
    assert np.array_equal(u32(got), u32(c.want()))


def test_attention_value_scores_out_of_range_are_reported(cuda_ok):
    errs()
    c = Case(5, 1, 1, 64, 32, [40], [[-1, 0]])
    c.q[...] = (1 << 24) - 1
    c.k[...] = (1 << 24) - 1
    c.upload().run()
    assert errs() & 16


def test_attention_equals_a_chain_of_smaller_calls(cuda_ok):
    """A node's bytes do not depend on the tree around it, the other sequences or the page size."""
    r = np.random.default_rng(4)
    t = tree(r, 40, 0.5)
    c = Case(9, 2, 2, 128, 64, [333], [t]).upload()
    whole = c.run().cpu().numpy()
    for i in (0, 7, 39):
        path = chain(t, i)
        one = Case(9, 2, 2, 128, 64, [333], [t])
        slots = 333 + np.arange(len(t))
        pg, off = one.tab[0, slots // 64], slots % 64
        one.k[pg[:len(path)], 0, :, off[:len(path)]] = one.k[pg[path], 0, :, off[path]]
        one.v[pg[:len(path)], 0, :, off[:len(path)]] = one.v[pg[path], 0, :, off[path]]
        one.trees, one.rows = [[j - 1 for j in range(len(path))]], len(path)
        one.q = one.q[path]
        one.row0, one.parent = np.array([0, len(path)], np.int32), np.arange(-1, len(path) - 1, dtype=np.int32)
        assert np.array_equal(u32(one.upload().run().cpu().numpy()[-1]), u32(whole[i]))


def test_attention_rows_out_of_range(cuda_ok):
    """A sequence whose arrays are out of range is reported and leaves its rows as they were; the others' are right."""
    r = np.random.default_rng(4)
    good = Case(21, 1, 2, 64, 32, [50, 60, 70], [tree(r, 5), tree(r, 6), tree(r, 7)]).upload()
    want = good.run().cpu().numpy()
    errs()

    def bad(name, at, value):
        old = good.d[name].clone()
        good.d[name].view(-1)[at] = value
        got = good.run(max_ctx=70).cpu().numpy()
        e = errs()
        good.d[name].copy_(old)
        return got, e

    for name, at, value, rows in (("ctx", 1, -1, (5, 11)), ("ctx", 1, 71, (5, 11)), ("ctx", 1, 1 << 30, (5, 11)),
                                  ("parent", 7, 2, (5, 11)), ("parent", 5, 0, (5, 11)), ("parent", 8, -2, (5, 11)),
                                  ("parent", 10, 1 << 30, (5, 11))):
        got, e = bad(name, at, value)
        assert e == 128, (name, at, value)
        keep = np.ones(18, bool)
        keep[rows[0]:rows[1]] = False
        assert np.array_equal(u32(got[keep]), u32(want[keep])) and (got[~keep] == 7.0).all(), (name, at, value)
    for value in (-1, 1000, 1 << 30, -(1 << 31)):
        got, e = bad("row0", 3, value)          # the last sequence's end: 18 -> out of range
        assert e == 128 and np.array_equal(u32(got[:11]), u32(want[:11])) and (got[11:] == 7.0).all()
    for value in (-1, 10 ** 6, -(1 << 31), (1 << 31) - 1):      # a page outside the pool: reported, nothing read there
        got, e = bad("tab", good.ld, value)
        assert e & 128 and np.array_equal(u32(got[:5]), u32(want[:5])) and np.array_equal(u32(got[11:]), u32(want[11:]))


def test_attention_rows_behind_the_last_sequence(cuda_ok):
    c = Case(2, 1, 2, 64, 32, [20], [tree(np.random.default_rng(0), 6)]).upload()
    want = c.run().cpu().numpy()
    c.d["row0"][1] = 4
    got = c.run().cpu().numpy()
    assert np.array_equal(u32(got[:4]), u32(want[:4])) and (got[4:] == 7.0).all()


def test_attention_far_pages(cuda_ok):
    """Page offsets beyond 2^32 bytes and 2^31 elements."""
    NKV, HD, page, layers = 4, 256, 4096, 3
    n_pages = 171                                            # 171 * 3 * 4 * 4096 * 256 elements > 2^31
    k = torch.zeros((n_pages, layers, NKV, page, HD), dtype=torch.int32, device="cuda")
    v = torch.zeros_like(k)
    c = Case(8, NKV, 2, HD, page, [45], [tree(np.random.default_rng(3), 7)], layers=layers, layer=2, spare=0)
    k[n_pages - 1] = dev(c.k[c.tab[0, 0]])
    v[n_pages - 1] = dev(c.v[c.tab[0, 0]])
    want = c.want()
    c.upload()
    c.d["tab"].fill_(n_pages - 1)
    c.view.k, c.view.v, c.view.n_pages = k.data_ptr(), v.data_ptr(), n_pages
    assert np.array_equal(u32(c.run().cpu().numpy()), u32(want))


def test_attention_streams_and_graphs(cuda_ok):
    """Two streams at once, and two captured graphs replayed at once: no shared workspace."""
    L = spb200.load()
    r = np.random.default_rng(6)
    cs = [Case(31 + i, 2, 2, 128, 64, [400 + 100 * i], [tree(r, 12 + i)]).upload() for i in range(2)]
    want = [c.run().cpu().numpy() for c in cs]
    st = [torch.cuda.Stream() for _ in cs]
    outs = [torch.zeros(w.shape, device="cuda") for w in want]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s, o in zip(cs, st, outs):
            c.run(out=o, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(np.array_equal(u32(o.cpu().numpy()), u32(w)) for o, w in zip(outs, want))
    graphs = []
    for c, s, o in zip(cs, st, outs):
        o.zero_()
        torch.cuda.synchronize()
        g = C.c_void_p()
        spb200.check(L.spb_graph_begin(s.cuda_stream))
        c.run(out=o, stream=s.cuda_stream)
        spb200.check(L.spb_graph_end(s.cuda_stream, C.byref(g)))
        graphs.append(g)
    for _ in range(10):
        for g, s in zip(graphs, st):
            spb200.check(L.spb_graph_launch(g, s.cuda_stream))
    torch.cuda.synchronize()
    assert all(np.array_equal(u32(o.cpu().numpy()), u32(w)) for o, w in zip(outs, want))
    for g in graphs:
        L.spb_graph_free(g)


# ------------------------------------------------------------------------------ compaction
@pytest.mark.parametrize("HD,page,ctx,paths", [
    (64, 128, [0], [[0]]),
    (64, 16, [10], [[0, 2, 5, 6, 9]]),
    (128, 24, [23, 100], [[1, 2, 3], [0, 1, 2]]),                       # a shift by one; in place already
    (256, 7, [3, 50, 9], [[63], list(range(1, 64)), []]),               # the last slot; a run as long as can be; none
    (64, 128, [120], [[1, 3, 5, 7, 9, 11, 13, 15, 17, 19, 40, 41]]),    # across a page
])
def test_compact_moves_the_path(cuda_ok, HD, page, ctx, paths):
    errs()
    c = Case(17, 2, 1, HD, page, ctx, [[-1] * 64 for _ in ctx], layers=3).upload()
    wk, wv = c.k.copy(), c.v.copy()
    for b, p in enumerate(paths):
        at = lambda slots: (c.tab[b, np.array(slots, int) // page], np.array(slots, int) % page)  # noqa: E731
        (sp, so), (dp, do) = at([ctx[b] + i for i in p]), at([ctx[b] + i for i in range(len(p))])
        for w in (wk, wv):
            w[dp, :, :, do] = w[sp, :, :, so]
    p0, p = dev(np.cumsum([0] + [len(x) for x in paths]).astype(np.int32)), dev(np.array(sum(paths, []), np.int32))
    spb200.kv_compact(c.view, len(ctx), c.d["ctx"].data_ptr(), p0.data_ptr(), p.data_ptr(), p.numel())
    assert np.array_equal(c.d["k"].cpu().numpy(), wk) and np.array_equal(c.d["v"].cpu().numpy(), wv)
    assert errs() == 0


@pytest.mark.parametrize("path", [[0, 2, 2], [3, 1], [-1, 4], [0, 64], [0, 1 << 30]])
def test_compact_refuses_a_bad_path(cuda_ok, path):
    errs()
    c = Case(17, 2, 1, 64, 16, [30, 40], [[-1] * 20, [-1] * 20], layers=2).upload()
    p0, p = dev(np.array([0, len(path), len(path) + 1], np.int32)), dev(np.array(path + [3], np.int32))
    spb200.kv_compact(c.view, 2, c.d["ctx"].data_ptr(), p0.data_ptr(), p.data_ptr(), p.numel())
    assert errs() == 128
    wk = c.k.copy()
    wk[c.tab[1, 40 // 16], :, :, 40 % 16] = wk[c.tab[1, 43 // 16], :, :, 43 % 16]   # the other sequence's moved
    assert np.array_equal(c.d["k"].cpu().numpy(), wk)


def test_compact_refuses_slots_and_pages_outside(cuda_ok):
    c = Case(17, 1, 1, 64, 16, [30], [[-1] * 20]).upload()
    p0, p = dev(np.array([0, 2], np.int32)), dev(np.array([0, 40], np.int32))     # slot 70 of a 64-slot table
    errs()
    spb200.kv_compact(c.view, 1, c.d["ctx"].data_ptr(), p0.data_ptr(), p.data_ptr(), 2)
    assert errs() == 128
    p[1] = 19
    for value in (-1, c.k.shape[0], 1 << 30):
        c.d["tab"][0, 49 // 16] = value
        spb200.kv_compact(c.view, 1, c.d["ctx"].data_ptr(), p0.data_ptr(), p.data_ptr(), 2)
        assert errs() == 128
    assert np.array_equal(c.d["k"].cpu().numpy(), c.k)


# ------------------------------------------------------------------------------ log probabilities
def lp_ref(x, tok_row, tok, top):
    """64-bit; ids by value, then lowest id; ids -1 / -inf where no entry above -inf is left."""
    x = x.astype(np.float64)
    m = x.max(1)
    with np.errstate(invalid="ignore", divide="ignore"):
        d = np.where(np.isneginf(x), -np.inf, x - np.where(np.isfinite(m), m, 0.0)[:, None])
        e = np.exp(d)
        s = e.sum(1)
        lse = m + np.log(s)
        ent = np.log(s) - np.where(e > 0, e * np.where(e > 0, d, 0.0), 0.0).sum(1) / s
    lse[np.isneginf(m)], ent[np.isneginf(m)] = -np.inf, 0.0
    bad = ~(x < np.inf).all(1)
    lse[bad] = ent[bad] = np.nan
    ids, best = np.full((len(x), top), -1, np.int64), np.full((len(x), top), -np.inf)
    for r in range(len(x)):
        if bad[r]:
            best[r] = np.nan
            continue
        o = np.lexsort((np.arange(x.shape[1]), -x[r]))[:top]
        o = o[x[r, o] > -np.inf]
        ids[r, :len(o)], best[r, :len(o)] = o, x[r, o] - lse[r]
    lp = np.full(len(tok), np.nan)
    for i, (r, t) in enumerate(zip(tok_row, tok)):
        if 0 <= r < len(x) and 0 <= t < x.shape[1] and not bad[r]:
            lp[i] = -np.inf if np.isneginf(x[r, t]) else x[r, t] - lse[r]
    # differences below f32's lowest value (-3e38 - 3e38) have no f32 but -inf
    lp[lp < -3.4028236e38], best[best < -3.4028236e38] = -np.inf, -np.inf
    return lp, lse, ent, ids, best


def lp_tol(x, vocab):
    """Roundings, each of at most 2^-24 of its value (u): an exponential within 2 ulp (4 u) of an argument
    rounded once (u |x - m|, at most 20 u where e is worth counting: beyond it e < 2^-28 and its share is
    below u), partial sums added in a chain of at most C steps. So the sum is off by (C + 25) u relative and
    the logarithm by as much absolute, plus its own rounding and that of m + log, x - lse: 4 u (|m| + 20).
    The entropy's second sum holds terms e |d| of at most the entropy plus log sum in weight, off likewise."""
    u = 2.0 ** -24
    fin = np.abs(np.where(np.isfinite(x), x, 0.0)).max(1).astype(np.float64)   # one tolerance per row
    C = vocab / 256 + 64
    return u * (C + 25 + 4 * (fin + 20)), np.full(len(x), u * (2 * (C + 45) * 16 + 200))


def run_lp(x, tok_row, tok, top, ld=None, lse=True, ent=True):
    rows, vocab = x.shape
    ld = ld or vocab
    buf = np.full((rows, ld), 1e30, np.float32)
    buf[:, :vocab] = x
    d = dev(buf)
    dr, dt = dev(np.array(tok_row, np.int32)), dev(np.array(tok, np.int32))
    lp = torch.full((max(1, len(tok)),), 7.0, device="cuda")
    a, b = torch.full((rows,), 7.0, device="cuda"), torch.full((rows,), 7.0, device="cuda")
    ids, best = torch.full((rows, top), 7, dtype=torch.int32, device="cuda"), torch.full((rows, top), 7.0, device="cuda")
    spb200.logprobs(d.data_ptr(), rows, vocab, ld, dr.data_ptr() if len(tok) else None, dt.data_ptr() if len(tok) else None, len(tok),
                    lp.data_ptr(), a.data_ptr() if lse else None, b.data_ptr() if ent else None, top,
                    ids.data_ptr() if top else None, best.data_ptr() if top else None)
    return [t.cpu().numpy() for t in (lp[:len(tok)], a, b, ids, best)]


def near(got, want, tol):
    f = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~f & ~np.isnan(want)], want[~f & ~np.isnan(want)])
    tol = np.broadcast_to(tol if np.ndim(got) < 2 else tol[:, None], got.shape)
    off = np.abs(got[f].astype(np.float64) - want[f])
    assert (off <= tol[f]).all(), off.max()


def check_lp(x, tok_row, tok, top, **kw):
    got, want = run_lp(x, tok_row, tok, top, **kw), lp_ref(x, tok_row, tok, top)
    tol, tol_e = lp_tol(x, x.shape[1])
    near(got[0], want[0], tol[list(tok_row)])
    near(got[1], want[1], tol)
    near(got[2], want[2], tol_e)
    assert np.array_equal(got[3], want[3])
    near(got[4], want[4], tol)
    return got


@pytest.mark.parametrize("rows,vocab,top,pad", [
    (1, 1, 1, 0), (1, 2, 5, 0), (3, 31, 32, 1), (2, 1000, 0, 0), (5, 1025, 7, 3), (4, 4097, 20, 2), (64, 8192, 5, 0),
    (2, 151936, 32, 0), (3, 262144, 20, 0), (2, 262145, 1, 1), (150, 777, 3, 5),
])
def test_logprobs(cuda_ok, rows, vocab, top, pad):
    errs()
    r = np.random.default_rng(rows * 7 + vocab)
    x = (r.standard_normal((rows, vocab)) * 3).astype(np.float32)
    x[r.random(x.shape) < 0.1] = -np.inf
    tok_row = r.integers(0, rows, 2 * rows + 1)
    check_lp(x, tok_row, r.integers(0, vocab, 2 * rows + 1), top, ld=vocab + pad)
    assert errs() == 0


def test_logprobs_ties_and_order(cuda_ok):
    """Equal entries, lowest id first: constant rows, -0 and +0, few distinct values, sorted rows, one value far off."""
    V = 20000
    r = np.random.default_rng(1)
    x = np.stack([np.zeros(V), np.where(np.arange(V) % 2, -0.0, 0.0), r.integers(-2, 3, V), np.arange(V) / 1000.0,
                  -np.arange(V) / 1000.0, np.where(np.arange(V) == V - 1, 80.0, -80.0), np.where(np.arange(V) % 64 < 32, 3.0, 2.0),
                  (np.arange(V) % 4096 < 8) * 1.0]).astype(np.float32)
    check_lp(x, range(len(x)), [5] * len(x), 32)


def test_logprobs_crowded_rows(cuda_ok):
    """Large entries that crowd into few threads' groups, and great numbers of equal ones: the list of candidates
    overflows. Few distinct values (as logits that came from 8 bits), whole rows of one value, -inf in between."""
    V, r = 40003, np.random.default_rng(8)
    x = np.tile(r.standard_normal(V).astype(np.float32), (310, 1))
    x[:100, (np.arange(V) // 4) % 512 < 20] += 50.0
    x[100:200] = np.rint(x[100:200] * 2)
    x[200:300] = 1.25
    x[300:] = np.where(np.arange(V) % 3 == 0, -np.inf, 2.0)
    pick = [0, 99, 100, 200, 309]
    got = run_lp(x, range(310), [7] * 310, 32)
    want = lp_ref(x[pick], range(5), [7] * 5, 32)
    tol, tol_e = lp_tol(x[pick], V)
    for k, (g, w) in enumerate(zip(got, want)):
        if k == 3:
            assert np.array_equal(g[pick], w)
        else:
            near(g[pick], w, tol_e if k == 2 else tol)
    assert np.array_equal(u32(got[4][0]), u32(got[4][50])) and np.array_equal(got[3][0], got[3][50])


def test_logprobs_steep_rows(cuda_ok):
    """Entries that rise by steps along the row (the running reference moves), and values near f32's ends."""
    V = 70001
    x = np.stack([np.linspace(-300, 300, V), np.linspace(300, -300, V), np.where(np.arange(V) == V - 1, 3e38, -3e38),
                  np.full(V, -3.4e38), np.where(np.arange(V) % 1000 == 999, 1e37, 0.0), np.full(V, 2e37)]).astype(np.float32)
    check_lp(x, range(len(x)), [V - 1] * len(x), 3)


def test_logprobs_empty_and_broken_rows(cuda_ok):
    """Rows masked whole, all but one, by the lowest value, rows with NaN and with +inf; tokens of masked places."""
    V = 3001
    r = np.random.default_rng(2)
    x = r.standard_normal((8, V)).astype(np.float32)
    x[0] = -np.inf
    x[1], x[1, 77] = -np.inf, 2.5
    x[2] = np.finfo(np.float32).min
    x[3, 100] = np.nan
    x[4, 2999] = np.inf
    x[5, :2990] = -np.inf
    x[6, 0] = np.finfo(np.float32).max
    errs()
    check_lp(x, list(range(8)) * 2, [9] * 8 + [77] * 8, 20)
    assert errs() == 0
    got = run_lp(x, [7, -1, 8, 7, 7, 7], [-1, 5, 5, V, -2, 5], 0)
    assert np.isnan(got[0][:5]).all() and np.isfinite(got[0][5]) and errs() == 32


def test_logprobs_rows_do_not_depend_on_each_other(cuda_ok):
    """The same bytes for a row alone, among many, at another alignment, and in a wider buffer."""
    V = 50001
    r = np.random.default_rng(3)
    x = (r.standard_normal((40, V)) * 2).astype(np.float32)
    many = run_lp(x, range(40), [11] * 40, 9)
    for i in (0, 17, 39):
        one = run_lp(x[i:i + 1], [0], [11], 9, ld=V + 3)
        assert all(np.array_equal(u32(a[0]), u32(b[i])) for a, b in zip(one, many))


def test_logprobs_optional_outputs(cuda_ok):
    x = np.random.default_rng(4).standard_normal((3, 500)).astype(np.float32)
    got = run_lp(x, [], [], 0, lse=False)
    assert (got[1] == 7.0).all() and np.isfinite(got[2]).all()
    got = run_lp(x, [1], [3], 0, ent=False)
    assert (got[2] == 7.0).all() and np.isfinite(got[1]).all()


@pytest.mark.parametrize("rows,n_tok", [(700, 700), (700, 3), (9, 9), (1, 1), (2, 0)])
def test_logprobs_token_of_its_row(cuda_ok, rows, n_tok):
    """Without tok_row, token t is row t's; fewer tokens than rows leave the rest alone."""
    V = 997
    r = np.random.default_rng(5)
    x = (r.standard_normal((rows, V)) * 2).astype(np.float32)
    tok = r.integers(0, V, max(n_tok, 1)).astype(np.int32)
    if n_tok > 2:
        tok[1], tok[2] = -1, V
    d, t, lp = dev(x), dev(tok), torch.full((max(rows, 1),), 7.0, device="cuda")
    errs()
    spb200.logprobs(d.data_ptr(), rows, V, V, None, t.data_ptr(), n_tok, lp.data_ptr(), None, None, 0, None, None)
    got, want = lp.cpu().numpy(), lp_ref(x[:n_tok], range(n_tok), tok[:n_tok], 0)[0] if n_tok else np.zeros(0)
    near(got[:n_tok], want, lp_tol(x[:n_tok], V)[0] if n_tok else np.zeros(0))
    assert (got[n_tok:] == 7.0).all() and errs() == (32 if n_tok > 2 else 0)


def test_logprobs_many_tokens_of_few_rows(cuda_ok):
    """More tokens than a row's threads, some of them twice."""
    r = np.random.default_rng(6)
    x = (r.standard_normal((3, 40000)) * 2).astype(np.float32)
    tok_row, tok = r.integers(0, 3, 5000), r.integers(0, 40000, 5000)
    tok_row[100:200], tok[100:200] = 1, 17
    got = check_lp(x, tok_row, tok, 2)
    assert len(set(u32(got[0][100:200]).tolist())) == 1


def test_logprobs_and_moves_streams_and_graphs(cuda_ok):
    """Two streams at once, then two captured graphs of attention, scoring and the move, replayed at once; the
    graphs read what their buffers hold at each replay."""
    L = spb200.load()
    r = np.random.default_rng(12)
    jobs = []
    for i in range(2):
        n, V = 9 + i, 33000 + 7 * i
        c = Case(51 + i, 2, 2, 64, 32, [150 + 60 * i], [[-1] + list(range(n - 1))], layers=2, layer=1).upload()
        x = (r.standard_normal((n, V)) * 3).astype(np.float32)
        path = [0, 2, 3, 6, 8]
        j = dict(c=c, x=x, V=V, n=n, d=dev(x), tok=dev(np.arange(n, dtype=np.int32)), p0=dev(np.array([0, 5], np.int32)),
                 p=dev(np.array(path, np.int32)), lp=torch.zeros(n, device="cuda"), e=torch.zeros(n, device="cuda"),
                 ids=torch.zeros((n, 6), dtype=torch.int32, device="cuda"), best=torch.zeros((n, 6), device="cuda"),
                 out=torch.zeros((n, 256), device="cuda"), st=torch.cuda.Stream(), path=path)
        jobs.append(j)

    def score(j, st):
        spb200.logprobs(j["d"].data_ptr(), j["n"], j["V"], j["V"], None, j["tok"].data_ptr(), j["n"], j["lp"].data_ptr(), None,
                        j["e"].data_ptr(), 6, j["ids"].data_ptr(), j["best"].data_ptr(), st)

    def check(j):
        w = lp_ref(j["x"], range(j["n"]), range(j["n"]), 6)
        t, te = lp_tol(j["x"], j["V"])
        near(j["lp"].cpu().numpy(), w[0], t)
        near(j["e"].cpu().numpy(), w[2], te)
        assert np.array_equal(j["ids"].cpu().numpy(), w[3])
        near(j["best"].cpu().numpy(), w[4], t)

    for j in jobs:
        score(j, None)
        j["c"].run(out=j["out"])
        j["want"] = j["out"].cpu().numpy()
        check(j)
        j["ids"].zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for j in jobs:
            score(j, j["st"].cuda_stream)
    torch.cuda.synchronize()
    graphs = []
    for j in jobs:
        check(j)
        s, c, g = j["st"].cuda_stream, j["c"], C.c_void_p()
        j["out"].zero_()
        torch.cuda.synchronize()
        spb200.check(L.spb_graph_begin(s))
        c.run(out=j["out"], stream=s)
        score(j, s)
        spb200.kv_compact(c.view, 1, c.d["ctx"].data_ptr(), j["p0"].data_ptr(), j["p"].data_ptr(), 5, s)
        spb200.check(L.spb_graph_end(s, C.byref(g)))
        graphs.append(g)
    for rep in range(2):
        if rep:   # other inputs in the same buffers
            for j in jobs:
                j["x"] = j["x"][::-1].copy()
                j["d"].copy_(dev(j["x"]))
                j["c"].d["k"].copy_(dev(j["c"].k))
                j["c"].d["v"].copy_(dev(j["c"].v))
            torch.cuda.synchronize()
        for j, g in zip(jobs, graphs):
            spb200.check(L.spb_graph_launch(g, j["st"].cuda_stream))
        torch.cuda.synchronize()
        for j in jobs:
            check(j)
            assert np.array_equal(u32(j["out"].cpu().numpy()), u32(j["want"]))
            c = j["c"]
            wk = c.k.copy()
            for i, p in enumerate(j["path"]):
                a, b = c.ctx[0] + p, c.ctx[0] + i
                wk[c.tab[0, b // 32], :, :, b % 32] = wk[c.tab[0, a // 32], :, :, a % 32]
            assert np.array_equal(c.d["k"].cpu().numpy(), wk)
    for g in graphs:
        L.spb_graph_free(g)


@pytest.mark.parametrize("B", [33, 70])
def test_attention_and_moves_of_many_sequences(cuda_ok, B):
    """More sequences than a warp's lanes, some without nodes, in a padded batch whose last rows belong to none."""
    r = np.random.default_rng(B)
    ctx = [int(x) for x in r.integers(0, 90, B)]
    trees = [tree(r, int(n)) for n in r.integers(0, 5, B)]
    trees[0] = trees[B - 1] = []
    c = Case(61, 1, 3, 64, 16, ctx, trees).upload()
    want, rows = c.want(win=20), c.rows
    c.d["q"] = torch.cat([c.d["q"], torch.full((6, 192), 1 << 23, dtype=torch.int32, device="cuda")])
    c.d["parent"] = torch.cat([c.d["parent"], torch.full((6,), 99, dtype=torch.int32, device="cuda")])
    c.rows = rows + 6
    errs()
    got = c.run(win=20).cpu().numpy()
    assert np.array_equal(u32(got[:rows]), u32(want)) and (got[rows:] == 7.0).all() and errs() == 0
    paths = [list(range(len(t)))[len(t) % 2:] for t in trees]   # every other one shifts by one
    p0, p = dev(np.cumsum([0] + [len(x) for x in paths]).astype(np.int32)), dev(np.array(sum(paths, []), np.int32))
    spb200.kv_compact(c.view, B, c.d["ctx"].data_ptr(), p0.data_ptr(), p.data_ptr(), p.numel())
    wk = c.k.copy()
    for b, q in enumerate(paths):
        for i, n in enumerate(q):
            s, t = ctx[b] + n, ctx[b] + i
            wk[c.tab[b, t // 16], :, :, t % 16] = wk[c.tab[b, s // 16], :, :, s % 16]
    assert np.array_equal(c.d["k"].cpu().numpy(), wk) and errs() == 0


def test_attention_far_positions(cuda_ok):
    """A window behind 2^29 and 2^30 - 70 positions of a page table that names two pages again and again."""
    page, n, win = 8192, 9, 300
    c = Case(81, 2, 2, 64, page, [page - n, page - n], [tree(np.random.default_rng(4), n)] * 2, spare=0).upload()
    ctx = [(1 << 29) + 77, (1 << 30) - 70]
    tab = torch.zeros((2, (1 << 30) // page), dtype=torch.int32, device="cuda")
    tab[0, 0::2], tab[0, 1::2] = int(c.tab[0, 0]), int(c.tab[1, 0])
    tab[1, 0::2], tab[1, 1::2] = int(c.tab[1, 0]), int(c.tab[0, 0])
    c.d["ctx"], c.view.ptab, c.view.ptab_ld = dev(np.array(ctx, np.int32)), tab.data_ptr(), tab.shape[1]
    errs()
    got = c.run(win=win, max_ctx=1 << 30).cpu().numpy()
    assert errs() == 0
    want = []
    for b in range(2):
        slots = np.arange(ctx[b] - win, ctx[b] + n)   # nothing before them is visible
        pg = tab[b].cpu().numpy()[slots // page]
        want.append(attend(c.k[pg, 0, :, slots % page], c.v[pg, 0, :, slots % page], c.q[n * b:n * b + n], win, c.trees[b], win, 2))
    assert np.array_equal(u32(got), u32(np.concatenate(want)))


@pytest.mark.parametrize("G,HD,win", [(3, 64, 7), (5, 128, 40), (6, 64, 1), (7, 64, 100), (8, 128, 33)])
def test_attention_tiles_inside_a_nodes_heads(cuda_ok, G, HD, win):
    """16 query vectors begin inside a node's heads; windows shorter and longer than the tree is deep."""
    c = Case(71, 2, G, HD, 24, [61], [tree(np.random.default_rng(G), 23, 0.8)]).upload()
    assert np.array_equal(u32(c.run(win=win).cpu().numpy()), u32(c.want(win=win)))


def test_odd_addresses_are_refused(cuda_ok):
    """Device pointers off a 4-byte boundary come back as an error (the host refuses them: nothing runs)."""
    c = Case(9, 1, 1, 64, 16, [20], [[-1, 0]]).upload()
    d, v = {n: t.data_ptr() for n, t in c.d.items()}, c.view
    out = torch.zeros(2, 64, device="cuda").data_ptr()
    args = [d["ctx"], d["row0"], d["parent"], out]
    for i in range(4):
        a = [p + 2 * (i == j) for j, p in enumerate(args)]
        with pytest.raises(spb200.SpbError):
            spb200.tree_attn(v, 0, 1, a[0], a[1], a[2], 2, 20, d["q"], 1, -1, a[3])
        if i < 3:
            with pytest.raises(spb200.SpbError):
                spb200.kv_compact(v, 1, a[0], a[1], a[2], 2)
    v.ptab += 1
    with pytest.raises(spb200.SpbError):
        spb200.kv_compact(v, 1, d["ctx"], d["row0"], d["parent"], 2)
    x, i32 = torch.zeros(4, 64, device="cuda").data_ptr(), torch.zeros(64, dtype=torch.int32, device="cuda").data_ptr()
    args = [x, i32, i32, x, x, x, i32, x]
    for i in range(8):
        a = [p + (i == j) for j, p in enumerate(args)]
        with pytest.raises(spb200.SpbError):
            spb200.logprobs(a[0], 2, 64, 64, a[1], a[2], 2, a[3], a[4], a[5], 3, a[6], a[7])


# ------------------------------------------------------------------------------ the whole step
@pytest.fixture(scope="module", params=["micro_gemma", "micro_qwen"])
def env(request):
    cfg = spmodel.CONFIGS[request.param]
    T = spmodel.gen_model(cfg, seed=5)
    m = spb200.Model.upload(cfg, T)
    pool = spb200.KvPool(m, 128, 48)
    yield cfg, T, m, pool
    pool.free()
    m.free()


def softmax_lp(row, tok):
    row = row.astype(np.float64)
    return row[tok] - (row.max() + np.log(np.exp(row - row.max()).sum()))


def check_tree(xs, xlast, toks, parent, res, V):
    """Every node's logits are XREF's on a clone that decodes the path; logprobs follow from XREF's rows."""
    rows = {}
    for i in range(len(parent)):
        s = xs.clone()
        for j in chain(parent, i):
            row = s.step(int(toks[j]))
        s.close()
        rows[i] = row
        assert np.array_equal(u32(res.logits[i]), u32(row)), i
        assert res.argmax[i] == int(row.argmax())
    tol = lp_tol(np.stack([rows[i] for i in range(len(parent))]), V)[0]
    for i, p in enumerate(parent):
        if p < 0:
            assert np.isnan(res.logprob[i])
        else:
            assert abs(res.logprob[i] - softmax_lp(rows[p], int(toks[i]))) <= tol[p]
    return rows


@pytest.mark.parametrize("paged", [False, True])
def test_tree_step_and_commit(xr, cuda_ok, env, paged):
    """Trees over a growing context (it crosses a page and the sliding window), commits of several paths, decoding on."""
    cfg, T, m, pool = env
    r = np.random.default_rng(12)
    pmax = 190
    s = pool.session(pmax) if paged else m.session(pmax)
    xs = xr.session(xref.build_desc(cfg, T), pmax)
    prompt = spmodel.gen_tokens(3, 110, cfg.n_vocab)
    s.prefill(prompt, logits=False)
    xs.prefill(prompt, all_logits=False)
    for n, accept in ((1, 1), (9, 3), (20, 2), (6, 0), (12, 4)):
        parent = tree(r, n, 0.6)
        toks = r.integers(0, cfg.n_vocab, n)
        res = s.tree_step(toks, parent, top=4)
        assert s.position() == xs.position()
        rows = check_tree(xs, None, toks, parent, res, cfg.n_vocab)
        for i in range(n):
            o = np.lexsort((np.arange(cfg.n_vocab), -rows[i]))[:4]
            assert np.array_equal(res.top_id[i], o)
        deepest = max(range(n), key=lambda i: len(chain(parent, i)))
        path = chain(parent, deepest)[:accept]
        s.tree_commit(path)
        for j in path:
            xs.step(int(toks[j]))
        assert s.position() == xs.position()
        for L in (0, cfg.n_layers - 1):
            for p in range(s.position() - len(path), s.position()):
                assert np.array_equal(s.kv(L, p, 0), xs.kv(L, p, 0)) and np.array_equal(s.kv(L, p, 1), xs.kv(L, p, 1))
        tok = int(r.integers(0, cfg.n_vocab))
        assert np.array_equal(u32(s.step(tok)), u32(xs.step(tok)))
    s.close()
    xs.close()


def test_tree_batch_of_sessions(xr, cuda_ok, env):
    """Paged and unpaged sessions with trees of their own in one step; 64 nodes in all."""
    cfg, T, m, pool = env
    r = np.random.default_rng(13)
    ss, xss, trees, toks = [], [], [], []
    for b, (ctx, n) in enumerate([(5, 1), (130, 31), (17, 12), (64, 20)]):
        s = pool.session(170) if b % 2 else m.session(170)
        x = xr.session(xref.build_desc(cfg, T), 170)
        p = spmodel.gen_tokens(20 + b, ctx, cfg.n_vocab)
        s.prefill(p, logits=False)
        x.prefill(p, all_logits=False)
        ss.append(s)
        xss.append(x)
        trees.append(tree(r, n, 0.5))
        toks.append(r.integers(0, cfg.n_vocab, n))
    res = spb200.batch_tree_step(ss, toks, trees, top=1)
    for x, t, p, o in zip(xss, toks, trees, res):
        check_tree(x, None, t, p, o, cfg.n_vocab)
    for s, p, x, t in zip(ss, trees, xss, toks):
        path = chain(p, len(p) - 1)
        s.tree_commit(path)
        for j in path:
            x.step(int(t[j]))
        assert np.array_equal(u32(s.step(3)), u32(x.step(3)))
    for s in ss + xss:
        s.close()


def test_tree_with_a_clone_between(xr, cuda_ok, env):
    """A paged clone taken while a tree is cached shares its pages: the commit copies before it moves rows."""
    cfg, T, m, pool = env
    s = pool.session(170)
    xs = xr.session(xref.build_desc(cfg, T), 170)
    prompt = spmodel.gen_tokens(30, 100, cfg.n_vocab)
    s.prefill(prompt, logits=False)
    xs.prefill(prompt, all_logits=False)
    s.tree_step([5, 6, 7, 8], [-1, -1, 1, 2], logits=False)
    c = s.clone()
    with pytest.raises(spb200.SpbError) as e:
        c.tree_commit([0])                       # the tree stays the original's
    assert e.value.code == spb200.SPB_EBADSTATE
    xc = xs.clone()
    s.tree_commit([1, 2, 3])
    for t in (6, 7, 8):
        xs.step(t)
    assert np.array_equal(u32(s.step(9)), u32(xs.step(9)))
    assert np.array_equal(u32(c.step(11)), u32(xc.step(11)))
    for x in (s, c, xs, xc):
        x.close()


def test_tree_states_and_refusals(cuda_ok, env):
    cfg, T, m, pool = env
    s = m.session(40)
    s.prefill([1, 2, 3], logits=False)

    def code(f):
        with pytest.raises(spb200.SpbError) as e:
            f()
        return e.value.code

    assert code(lambda: s.tree_commit([])) == spb200.SPB_EBADSTATE
    assert code(lambda: s.tree_step([1, 2], [-1, 1])) == spb200.SPB_EBADARG
    assert code(lambda: s.tree_step([1, 2], [-2, 0])) == spb200.SPB_EBADARG
    assert code(lambda: s.tree_step(list(range(38)), [-1] * 38)) == spb200.SPB_ECONTEXT_FULL
    assert code(lambda: s.tree_step([1] * 65, [-1] * 65)) == spb200.SPB_EBADARG
    assert code(lambda: s.tree_step([1], [-1], top=33)) == spb200.SPB_EBADARG
    assert code(lambda: s.tree_step([cfg.n_vocab], [-1])) == spb200.SPB_ERANGE
    assert code(lambda: spb200.batch_tree_step([s, s], [[1], [1]], [[-1], [-1]])) == spb200.SPB_EBADARG
    before = s.step(4)
    s.rewind(1)
    for spoil in (lambda: s.step(4), lambda: s.prefill([4], logits=False), lambda: s.greedy(4, 1),
                  lambda: spb200.batch_decode([s], [4]), lambda: s.score([4])):
        s.tree_step([1, 2, 3], [-1, 0, 0])
        assert code(lambda: s.tree_commit([1])) == spb200.SPB_EBADARG
        assert code(lambda: s.tree_commit([0, 2, 1])) == spb200.SPB_EBADARG
        assert code(lambda: s.tree_commit([3])) == spb200.SPB_EBADARG
        spoil()
        assert code(lambda: s.tree_commit([0])) == spb200.SPB_EBADSTATE
        s.rewind(1)
    s.tree_step([1, 2, 3], [-1, 0, 0])
    s.rewind(0)
    assert code(lambda: s.tree_commit([0])) == spb200.SPB_EBADSTATE
    assert np.array_equal(u32(s.step(4)), u32(before))      # none of it moved the context
    z = m.session(40, spinor=True)
    z.prefill([1, 2], logits=False)
    assert code(lambda: z.tree_step([1], [-1])) == spb200.SPB_EUNSUPPORTED
    z.close()
    s.close()


@pytest.mark.parametrize("n", [1, 2, 65, 150])
def test_score(xr, cuda_ok, env, n):
    """A prompt's log probabilities, entropies and alternatives against XREF's logits; the position moves as in a prefill."""
    cfg, T, m, pool = env
    s = m.session(200)
    xs = xr.session(xref.build_desc(cfg, T), 200)
    first = spmodel.gen_tokens(40, 20, cfg.n_vocab)
    s.prefill(first, logits=False)
    xs.prefill(first, all_logits=False)
    toks = spmodel.gen_tokens(41, n, cfg.n_vocab)
    res, rows = s.score(toks, top=3, logits=True), xs.prefill(toks)
    assert np.array_equal(u32(res.logits), u32(rows)) and s.position() == xs.position()
    tol, tol_e = lp_tol(rows, cfg.n_vocab)
    lp, _, ent, ids, best = lp_ref(rows, range(n - 1), toks[1:], 3)
    assert np.isnan(res.logprob[0])
    near(res.logprob[1:], lp, tol[:-1])
    near(res.entropy, ent, tol_e)
    assert np.array_equal(res.top_id, ids) and np.array_equal(res.argmax, ids[:, 0])
    near(res.top_logprob, best, tol)
    assert np.array_equal(u32(s.step(3)), u32(xs.step(3)))
    s.close()
    xs.close()


def test_score_long_and_in_pieces(xr, cuda_ok, env):
    """A whole chunk of 256 rows and its rest; pieces give the bytes of the whole, but for their first tokens."""
    cfg, T, m, pool = env
    n = 323
    s, xs = m.session(400), xr.session(xref.build_desc(cfg, T), 400)
    toks = spmodel.gen_tokens(43, n, cfg.n_vocab)
    res, rows = s.score(toks, top=3, logits=True), xs.prefill(toks)
    assert np.array_equal(u32(res.logits), u32(rows)) and s.position() == n
    tol, tol_e = lp_tol(rows, cfg.n_vocab)
    lp, _, ent, ids, best = lp_ref(rows, range(n - 1), toks[1:], 3)
    near(res.logprob[1:], lp, tol[:-1])
    near(res.entropy, ent, tol_e)
    assert np.array_equal(res.top_id, ids) and np.array_equal(res.argmax, rows.argmax(1))
    near(res.top_logprob, best, tol)
    s.rewind(n)
    at = 0
    for k in (1, 130, n - 131):
        part = s.score(toks[at:at + k], top=3)
        assert np.isnan(part.logprob[0]) and np.array_equal(u32(part.logprob[1:]), u32(res.logprob[at + 1:at + k]))
        assert np.array_equal(u32(part.entropy), u32(res.entropy[at:at + k])) and np.array_equal(part.top_id, res.top_id[at:at + k])
        at += k
    s.close()
    xs.close()
