"""Values at which the kernels that verify drafted trees can go wrong: every distance of a score below
its maximum, contexts that go in runs, logits of every magnitude, finite masks, peaked rows."""
import numpy as np
import pytest
import torch

import spb200
from test_gpu_tree import Case, chain, dev, errs, exp_fixed, run_lp, tree, u32

pytestmark = pytest.mark.gpu

ONE = 1 << 30
U = 2.0 ** -24                                             # half a step of f32, relative


# ------------------------------------------------------------------------------ attention
def test_attention_every_distance_below_the_maximum(cuda_ok):
    """A node sees one context slot of score 0 and itself, `far` grid steps (2^-14) below: with one column of
    q and k the score is exact. All distances up to 32 octaves (363408.75 steps) and past them."""
    HD, n = 64, 64
    far = np.concatenate([np.arange(0, 363600), np.exp(np.linspace(np.log(363600), np.log((1 << 24) - 1), 2000)).astype(np.int64)])
    far = np.concatenate([far, np.full(-len(far) % n, 1 << 19)])
    B, page = len(far) // n, n + 1
    r = np.random.default_rng(0)
    k, v = np.zeros((B, 1, 1, page, HD), np.int32), np.zeros((B, 1, 1, page, HD), np.int32)
    k[:, 0, 0, 1:, 0] = -far.reshape(B, n)
    value = r.integers(-(1 << 30) + 1, 1 << 30, HD)
    v[:, 0, 0, 1:] = value
    q = np.zeros((B * n, HD), np.int32)
    q[:, 0] = 1 << 21                                      # score -far 2^21 2^-32 / 8 = -far 2^-14
    d = [dev(a) for a in (k, v, np.ones(B, np.int32), np.arange(0, B * n + 1, n).astype(np.int32), np.full(B * n, -1, np.int32), q)]
    out = torch.full((B * n, HD), 7.0, device="cuda")
    view = spb200.KvView(d[0].data_ptr(), d[1].data_ptr(), None, B, page, 0, 1, 1, HD)
    errs()
    spb200.tree_attn(view, 0, B, d[2].data_ptr(), d[3].data_ptr(), d[4].data_ptr(), B * n, 1, d[5].data_ptr(), 1, -1, out.data_ptr())
    got = out.cpu().numpy()
    assert errs() == 0
    e = exp_fixed(far)[:, None]
    S, w = ONE + e, e * value[None, :]                     # floor(e v 2^16 / S), in two steps of int64
    want = (((w // S) << 16) + ((w % S) << 16) // S).astype(np.float64) * 2.0 ** -32
    wrong = (u32(got) != u32(want.astype(np.float32))).any(1)
    assert not wrong.any(), far[wrong]


# ------------------------------------------------------------------------------ log probabilities
def lp_exact(x, tok_row, tok, top):
    """64-bit, from differences to the row's maximum (x - lse would lose log(sum) to a maximum of 1e30)."""
    x = x.astype(np.float64)
    m = x.max(1, keepdims=True)
    d = np.maximum(x - m, -1e300)
    e = np.exp(d)
    s = e.sum(1)
    mean = (e * np.where(e > 0, d, 0.0)).sum(1) / s        # sum p (x - m)
    order = np.argsort(-x, axis=1, kind="stable")[:, :top]
    at = np.take_along_axis(x, order, 1)
    ids = np.where(at > -np.inf, order, -1)
    best = at - m - np.log(s)[:, None]
    lp = (x[tok_row, tok] - m[tok_row, 0]) - np.log(s)[tok_row]
    low = -3.4028236e38                                    # differences below f32's lowest value have no f32 but -inf
    return np.where(lp < low, -np.inf, lp), m[:, 0] + np.log(s), np.log(s) - mean, ids, np.where(best < low, -np.inf, best)


def lp_bounds(x):
    """How far log(sum), and the entropy, may be off; every rounding at most U of its value.

    An addend e = 2^((x - r) log2 e) of a thread's reference r: the exponential 4 U, its argument two roundings
    and the constant's (2.25 U |x - r|). Sums are moved to larger references at most N times (a thread's batches
    of 8192 entries, the warp, 16 warps by halves, 16 parts by halves): 4 U for the factor, 3 U for its use,
    U of the distance; the largest entry's own reference is the row's maximum: factors of 1, no error. Additions: as
    many as there are other entries above -inf, at most 16 in a batch, one a batch, 5 in the warp and the halvings'.
    The entropy's second sum has the same terms times their distance D (of one sign), a product and a shift of
    its own at every step."""
    x = x.astype(np.float64)
    m = x.max(1, keepdims=True)
    d = np.maximum(x - m, -1e300)
    e = np.exp(d)
    S = e.sum(1)
    p, D = e / S[:, None], np.where(e > 0, -d, 0.0)
    mean, sq = (p * D).sum(1), (p * D * D).sum(1)
    V = x.shape[1]
    parts = min(16, -(-V // 16384))
    batches = -(-(-(-V // parts) + 3) // 8192)
    N = batches + 10
    A = np.minimum(30 + batches, (x > -np.inf).sum(1) - 1)
    rel = (1 - p.max(1)) * (4 + 7 * N) + 3.25 * mean + A
    log = U * (rel + 2 * np.log(S))                        # (logf: one unit in its last place)
    ent = U * ((8 + 10 * N + 2 * A) * mean + 3.25 * sq + rel * mean + 4 * mean + 2 * (np.log(S) + mean))
    return log * 1.01 + 1e-38, (log + ent) * 1.01 + 1e-38  # (products of two errors)


def off(got, want, tol):
    f = np.isfinite(want)
    assert np.array_equal(got[~f], want[~f]), (got[~f], want[~f])
    d = np.abs(got[f].astype(np.float64) - want[f]) - np.broadcast_to(tol, want.shape)[f]
    assert (d <= 0).all(), (d.max(), np.argwhere(f)[d.argmax()], got[f][d.argmax()], want[f][d.argmax()])


def check_rows(x, tok, top=5, **kw):
    """Every row's log-sum-exp, entropy, alternatives and the log probabilities of the given columns."""
    x = x.astype(np.float32)
    rows = np.repeat(np.arange(len(x)), len(tok))
    tok = np.tile(np.asarray(tok), len(x))
    errs()
    got, want = run_lp(x, rows, tok, top, **kw), lp_exact(x, rows, tok, top)
    assert errs() == 0
    log, ent = lp_bounds(x)
    m = x.max(1).astype(np.float64)
    with np.errstate(invalid="ignore"):
        off(got[0], want[0], log[rows] + U * (np.abs(x[rows, tok] - m[rows]) + np.abs(want[0])))
        off(got[1], want[1], log + U * np.abs(want[1]))
        off(got[2], want[2], ent + U * np.abs(want[2]))
        assert np.array_equal(got[3], want[3])
        off(got[4], want[4], log[:, None] + U * (2 * np.abs(want[4]) + log[:, None] + np.log(len(x[0]))))
    assert (got[2] >= 0).all()


MASKS = [-1e4, -65504.0, -1e9, -10 ** 9.5, -1e10, -1e18, -1e20, -1e30, -1e36, float(np.finfo(np.float32).min)]


@pytest.mark.parametrize("V", [32000, 262144])
def test_logprobs_finite_masks(cuda_ok, V):
    """Masks written as large negative numbers, over half of a row, most of it, and its front or tail."""
    r = np.random.default_rng(1)
    x = []
    for mask in MASKS:
        for where in (r.random(V) < 0.5, r.random(V) < 0.9, np.arange(V) < V // 2, np.arange(V) >= V // 3, np.arange(V) != 777):
            x.append(np.where(where, mask, r.standard_normal(V) * 3))
    check_rows(np.stack(x), [777, V // 3 - 1, V - 1, 0])


def test_logprobs_rows_of_any_magnitude(cuda_ok):
    """Rows of one value, and ordinary rows around a far value, at every magnitude that f32 has."""
    V, r = 20011, np.random.default_rng(2)
    x = [np.full(V, s * 10.0 ** k) for k in (0, 2, 3, 3.6, 4, 5, 6, 7, 7.3, 8, 9, 9.5, 10, 12, 15, 20, 25, 30, 36, 37, 38) for s in (1, -1)]
    for c in (1e3, 4e3, 5e3, 1e4, 1e5, 1e6, 1e7, 3e7, 1e8, 1e9, 3e9):
        x += [r.standard_normal(V) * 3 + c, r.standard_normal(V) * 3 - c]
    for k in range(-6, 39, 2):                             # a spread of that size
        x.append(r.uniform(-1, 1, V) * 3 * 10.0 ** k)
    check_rows(np.stack(x), [0, 9999, V - 1], top=20)


def test_logprobs_two_entries_of_one_thread(cuda_ok):
    """A row of two entries, the second 0.5 to 17 above the first and 8192 columns behind it: the smaller came first,
    and what is left of the sum beside 1 is all that log(sum) and the entropy consist of."""
    V = 16384
    d = np.concatenate([np.linspace(0.5, 17, 200), [15.9, 15.95, 15.99]])
    x = np.full((len(d), V), -np.inf)
    x[:, 40], x[:, 40 + 8192] = 0.3, 0.3 + d
    check_rows(x, [40, 40 + 8192], top=3)


@pytest.mark.parametrize("V", [5000, 40001, 262144])
def test_logprobs_peaked_rows(cuda_ok, V):
    """One entry takes most of the row, anywhere in it; some of the others, or all, are far below."""
    r = np.random.default_rng(3)
    x = r.standard_normal((120, V))
    x[:40, r.random(V) < 0.9] = -np.inf
    x[40:80, r.random(V) < 0.9995] = -np.inf
    at = r.integers(0, V, 120)
    x[np.arange(120), at] = r.uniform(12, 16.9, 120)
    x[::2] += r.uniform(-300, 300, (60, 1))
    check_rows(x, [int(at[3]), int(at[50]), int(at[100]), 17], top=9)


def test_logprobs_rising_and_falling_rows(cuda_ok):
    """The maximum moves all along the row, by steps below and above 16."""
    V = 70001
    up = [np.linspace(-s, s, V) for s in (0.01, 1, 5, 12, 40, 300)]
    steps = [np.floor(np.arange(V) / 4096) * s for s in (0.3, 3.0, 15.9, 16.1, 40.0)]
    x = np.stack([y[::k] for y in up + steps for k in (1, -1)])
    check_rows(x, [0, V // 2, V - 1], top=4)


def attend_far(K, V, q, ctx, parent, win, G):
    """The contract (`attend`) for long contexts: V in digits of 10 bits, so that the sums fit int64."""
    n, NKV, HD = len(parent), K.shape[1], K.shape[2]
    asc = np.float32(1.0) / np.sqrt(np.float32(HD))
    out = np.zeros((n, NKV, G, HD), np.float32)
    for i in range(n):
        c = chain(parent, i)
        first = max(0, ctx + len(c) - win) if win > 0 else 0
        see = np.array(list(range(min(first, ctx), ctx)) + [ctx + a for t, a in enumerate(c) if ctx + t >= first])
        for g in range(NKV):
            k, v = K[see, g].astype(np.int64), V[see, g].astype(np.int64)
            v0, v1, v2 = v & 1023, (v >> 10) & 1023, v >> 20
            for h in range(G):
                s = (k * q[i].reshape(NKV, G, HD)[g, h].astype(np.int64)).sum(1)
                z = ((s.astype(np.float64) * 2.0 ** -32).astype(np.float32) * asc).astype(np.float64) * 16384.0
                zi = np.where(z < 0, np.ceil(z - 0.5), np.floor(z + 0.5)).astype(np.int64)
                e = exp_fixed(zi.max() - zi)
                S, N = int(e.sum()), [(e @ d).tolist() for d in (v0, v1, v2)]
                out[i, g, h] = [np.float32(float(((a + (b << 10) + (c2 << 20)) << 16) // S) * 2.0 ** -32) for a, b, c2 in zip(*N)]
    return out.reshape(n, NKV * G * HD)


def want_far(c, win=-1):
    res = []
    for b, ctx in enumerate(c.ctx):
        slots = np.arange(ctx + len(c.trees[b]))
        pg, at = c.tab[b, slots // c.page], slots % c.page
        res.append(attend_far(c.k[pg, c.layer, :, at], c.v[pg, c.layer, :, at], c.q[c.row0[b]:c.row0[b + 1]], ctx, c.trees[b], win, c.G))
    return np.concatenate(res)


def outliers(c):
    """Some entries at the grid's limits: their fourth digits are not zero."""
    lim = c.r.random(c.k.shape[:-1]) < 0.002
    c.k[lim, 3], c.v[lim, 5] = (1 << 24) - 1, -(1 << 30) + 1
    c.q[:, 3] = 1000
    return c


@pytest.mark.parametrize("HD,G,page,ctx,nodes", [
    (64, 2, 128, 34000, 3), (128, 1, 4096, 34000, 3), (256, 1, 128, 34000, 2), (64, 1, 1000, 70000, 3), (128, 2, 128, 70000, 2),
    (256, 1, 4096, 70000, 3),
])
def test_attention_in_runs(cuda_ok, HD, G, page, ctx, nodes):
    """More slots than a cluster of CTAs keeps scores for (16 x 2112): maxima first, then run after run."""
    c = outliers(Case(13, 1, G, HD, page, [ctx], [tree(np.random.default_rng(1), nodes, 0.7)])).upload()
    errs()
    got = c.run().cpu().numpy()
    assert errs() == 0
    assert np.array_equal(u32(got), u32(want_far(c)))


@pytest.mark.parametrize("HD", [64, 128, 256])
def test_attention_in_runs_of_ragged_sequences(cuda_ok, HD):
    """Long, short and empty contexts, and a sequence without nodes, in one call; 32 heads' worth of nodes."""
    r = np.random.default_rng(2)
    ctx, nodes = [500, 35001, 0, 1056, 77], [20, 2, 5, 0, 1]
    c = outliers(Case(14, 2, 2, HD, 96, ctx, [tree(r, n, 0.5) for n in nodes])).upload()
    assert np.array_equal(u32(c.run().cpu().numpy()), u32(want_far(c)))


@pytest.mark.parametrize("HD,win", [(64, 35000), (256, 34000)])
def test_attention_in_runs_of_a_window(cuda_ok, HD, win):
    c = outliers(Case(15, 1, 2, HD, 128, [40000], [[-1, 0, 1, -1]])).upload()
    assert np.array_equal(u32(c.run(win=win).cpu().numpy()), u32(want_far(c, win)))


@pytest.mark.parametrize("HD", [64, 128, 256])
@pytest.mark.parametrize("nodes,ctx", [(64, 300), (7, 5000)])
def test_attention_in_runs_or_not(cuda_ok, HD, nodes, ctx):
    """A call that allows for long contexts gives short ones the same bytes."""
    c = outliers(Case(16, 2, 2, HD, 64, [ctx, 40], [tree(np.random.default_rng(3), n, 0.6) for n in (nodes, 3)])).upload()
    one = c.run().cpu().numpy()
    for far in (33729, 200000, 1048512):
        assert np.array_equal(u32(c.run(max_ctx=far).cpu().numpy()), u32(one))
