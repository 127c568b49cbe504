"""The operators of speculative decoding with a tree of drafted tokens: real calls over the real range.

A drafter proposes a tree of tokens after every sequence's context. One step of the model then needs
  attention  every drafted token attends to the cached context and to its own ancestors in the tree,
  logprobs   the model's log probability of the drafted tokens, its entropy and its best alternatives,
  compact    once a path through the tree is accepted, its K and V rows move to the positions that follow
             the context, in every layer, inside the pages of the cache.
`run` is one call of one of them: with `own` false in plain torch operations, with `own` true as a user of
the framework calls it. Formulas:

Attention. q, k, v are integers on the 2^16 grid (|q|, |k| < 2^24, |v| < 2^30). Node i of a sequence with
context c and depth d (its number of ancestors) stands at position p = c + d and is cached in slot c + i.
It sees the context's positions j < c and the slots of its ancestors and itself; with a window w only those
at positions above p - w. Per head: s = <q, k> exactly; z = f32(s 2^-32) f32(HD^-1/2) in f32;
zi = z 2^14 rounded half away from zero; e = the framework's integer exponential of (zi - max zi) 2^-14 in
2^30 fixed point; out = sum e v / sum e 2^-16, rounded once to f32.

Logprobs. lse = log sum exp x over the row; logprob = x[token] - lse; entropy = sum p (lse - x); the k
largest entries with their ids, equal ones lowest id first. Entries of -inf are masked tokens.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

ONE = 1 << 30
LOG2E = 1549082005                                   # round(log2(e) 2^30)
EXP2 = (1073741824, 744261118, 257941248, 59597083, 10327387, 1431680, 165394)   # round(ln(2)^k / k! 2^30)
FAR = 1 << 19                                         # grid steps below the maximum where e is 0 for certain

# heads, KV heads, head width, layers: the 12B and 8B shapes of the benchmark and its tiny one
SHAPES = {"12b": (16, 8, 256, 48), "8b": (32, 8, 128, 36), "tiny": (8, 2, 64, 4)}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a greedy chat turn's second step: one short context, a chain of four drafts
        dict(name="tree_chain4_ctx100", op="attention", shape="12b", seqs=1, nodes=4, ctx=100, spread=0, window=-1, page=128),
        # a small model's odd-sized tree over pages that end inside a tile
        dict(name="tree_small_odd_pages", op="attention", shape="tiny", seqs=5, nodes=13, ctx=231, spread=1, window=-1, page=24),
        # sliding-window layers of the 12B shape behind the benchmark's 2048-token prompt
        dict(name="tree_window_16", op="attention", shape="12b", seqs=1, nodes=16, ctx=2050, spread=0, window=1024, page=4096),
        # the 8B shape at the benchmark's 4096-token prompt and a wide tree
        dict(name="tree_8b_31_ctx4133", op="attention", shape="8b", seqs=1, nodes=31, ctx=4133, spread=0, window=-1, page=128),
        # eight sessions of the speculative benchmark, ragged contexts up to 8192, eight drafts each
        dict(name="tree_8seq_8", op="attention", shape="12b", seqs=8, nodes=8, ctx=8192, spread=1, window=-1, page=128),
        # one long session verified with the largest tree
        dict(name="tree_64_ctx8192", op="attention", shape="12b", seqs=1, nodes=64, ctx=8192, spread=0, window=-1, page=128),
        # one decode row with its alternatives
        dict(name="lp_row_top5", op="logprobs", rows=1, vocab=262144, pad=0, top=5, masked=0.0, per_row=1),
        # a verified tree of 64 rows with alternatives, part of the vocabulary banned
        dict(name="lp_tree64_top20", op="logprobs", rows=64, vocab=262144, pad=0, top=20, masked=0.1, per_row=1),
        # a prompt scored: many rows, the 8B shape's vocabulary, entropies and no alternatives
        dict(name="lp_score_1000", op="logprobs", rows=1000, vocab=151936, pad=0, top=0, masked=0.0, per_row=1),
        # a vocabulary slice of odd length in a wider buffer, three candidates per row
        dict(name="lp_odd_slice", op="logprobs", rows=37, vocab=8191, pad=130, top=8, masked=0.3, per_row=3),
        # one session accepts a path of five nodes
        dict(name="compact_1seq_5", op="compact", shape="12b", seqs=1, nodes=32, accept=5, ctx=250, page=128),
        # eight sessions accept at once, their pages forked from one prompt
        dict(name="compact_8seq_12", op="compact", shape="8b", seqs=8, nodes=40, accept=12, ctx=300, page=128),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("attention", "attention", "logprobs", "compact"))
    if op == "attention":
        shape = rng.choice(("12b", "8b", "tiny"))
        seqs = rng.choice((1, 1, 2, 3, 5, 8))
        nodes = _log(rng, 1, 64 // seqs)
        spread = rng.randint(0, 1)
        return dict(op=op, shape=shape, seqs=seqs, nodes=nodes, ctx=_log(rng, 1, 8192 if spread or seqs < 3 else 4096), spread=spread,
                    window=rng.choice((-1, -1, 512, 1024)), page=rng.choice((24, 128, 128, 256, 8320)))
    if op == "logprobs":
        vocab = _log(rng, 500, 262144)
        top = rng.choice((0, 1, 5, 20, 32))
        rows = _log(rng, 1, min(1500, (15_000_000 if top else 150_000_000) // vocab))
        return dict(op=op, rows=rows, vocab=vocab, pad=rng.choice((0, 0, 1, 130)), top=top,
                    masked=rng.choice((0.0, 0.0, 0.2)), per_row=rng.choice((1, 1, 3)))
    nodes, seqs = rng.randint(4, 64), rng.choice((1, 2, 3))
    return dict(op=op, shape=rng.choice(("12b", "8b", "tiny")), seqs=seqs, nodes=nodes,
                accept=rng.randint(1, min(nodes // 2, 32 // seqs)), ctx=rng.randint(1, 330), page=128)


# ------------------------------------------------------------------------------------------ sizes
def _contexts(case, seed):
    """Every sequence's context: all of `ctx`, or one of `ctx` and the others uniform in [128, ctx]."""
    n, c = case["seqs"], case["ctx"]
    if not case["spread"]:
        return [c] * n
    r = np.random.RandomState(1)   # the same contexts for every seed: the case says what the work is
    return [c] + [int(r.randint(min(128, c), c + 1)) for _ in range(n - 1)]


def _visible(ctx, window):
    """Context positions that some node of the tree sees (the root's window reaches furthest back)."""
    return ctx if window < 0 else min(ctx, window - 1)


def work(case):
    if case["op"] == "attention":
        nh, nkv, hd, _ = SHAPES[case["shape"]]
        rows = case["seqs"] * case["nodes"]
        pos = sum(_visible(c, case["window"]) + case["nodes"] for c in _contexts(case, 0))
        pairs = sum(case["nodes"] * (_visible(c, case["window"]) + 1) for c in _contexts(case, 0))
        return {"bytes": 2 * pos * nkv * hd * 4 + 2 * rows * nh * hd * 4, "flops": 4 * pairs * nh * hd}
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        out = case["rows"] * (case["per_row"] * 12 + 8 + case["top"] * 8)
        return {"bytes": n * 4 + out, "flops": 5 * n}
    nh, nkv, hd, nl = SHAPES[case["shape"]]
    moved = case["seqs"] * case["accept"] * nl * nkv * hd
    return {"bytes": 2 * 2 * moved * 4, "flops": 0}


# ------------------------------------------------------------------------------------------ inputs
def _tree(r, n):
    """Parents of a drafted tree in the order of drafting: -1 for a first token, else an earlier node."""
    return [-1 if i == 0 or r.rand() < 0.1 else int(r.randint(max(0, i - 6), i)) for i in range(n)]


def _path(r, n, accept):
    """Accepted nodes in tree order: a first run already in place, then later ones (at or behind slot `accept`)."""
    keep = int(r.randint(0, accept + 1)) if n - accept >= accept else 0
    late = np.sort(r.choice(np.arange(accept, n), accept - keep, replace=False))
    return list(range(keep)) + [int(x) for x in late]


def _library():
    """The framework's package (its folder's name is no module name)."""
    if "spb200" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "shannon-prime-system_b200"))
    import spb200
    return spb200


def _pages(s):
    """The cache as the framework's calls take it: pools, page table and their sizes."""
    n, nl, nkv, page, hd = s["k"].shape
    return _library().KvView(s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(), n, page, s["table"].shape[1], nl, nkv, hd)


def _ints(x, lim):
    return (x * 65536.0).round_().clamp_(-lim, lim).to(torch.int32)


def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    r = np.random.RandomState(seed % (1 << 31))
    s = dict(case)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev) * scale

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    if case["op"] == "attention":
        nh, nkv, hd, _ = SHAPES[case["shape"]]
        B, T, page = case["seqs"], case["nodes"], case["page"]
        ctx = _contexts(case, seed)
        per = [-(-(c + T) // page) for c in ctx]                  # pages of each sequence
        n_pages, ld = sum(per) + 1, max(per)
        order, at, tab = r.permutation(n_pages), 0, np.zeros((B, ld), np.int32)
        for b in range(B):
            tab[b, :per[b]] = order[at:at + per[b]]
            at += per[b]
        s |= {"k": _ints(normal(n_pages, 1, nkv, page, hd), (1 << 24) - 1), "v": _ints(normal(n_pages, 1, nkv, page, hd), (1 << 24) - 1),
              "q": _ints(normal(B * T, nh * hd, scale=1.7), (1 << 24) - 1), "table": torch.from_numpy(tab).to(dev), "ctx": ints(ctx),
              "row0": ints([b * T for b in range(B + 1)]), "parent": ints(sum((_tree(r, T) for _ in range(B)), [])),
              "max_ctx": max(ctx), "out": torch.zeros(B * T, nh * hd, device=dev)}
    elif case["op"] == "logprobs":
        n, v = case["rows"], case["vocab"]
        x = normal(n, v + case["pad"], scale=2.5)
        x[:, :v].scatter_(1, torch.randint(0, v, (n, 4), generator=g, device=dev), 14.0 + normal(n, 4))
        if case["masked"]:
            x.masked_fill_(torch.rand(n, v + case["pad"], generator=g, device=dev) < case["masked"], -math.inf)
        m = n * case["per_row"]
        row = torch.arange(m, device=dev, dtype=torch.int32) // case["per_row"]
        # drafted tokens are likely ones: half of them among the row's best, the others anywhere
        best = x[:, :v].argmax(1)[row.long()].int()
        tok = torch.where(torch.rand(m, generator=g, device=dev) < 0.5, best, torch.randint(0, v, (m,), generator=g, device=dev).int())
        top = case["top"]
        s |= {"x": x, "row": row, "tok": tok.contiguous(), "logprob": torch.zeros(m, device=dev), "lse": torch.zeros(n, device=dev),
              "entropy": torch.zeros(n, device=dev), "ids": torch.zeros(n, top, dtype=torch.int32, device=dev),
              "best": torch.zeros(n, top, device=dev)}
    else:
        nh, nkv, hd, nl = SHAPES[case["shape"]]
        B, T, page, c = case["seqs"], case["nodes"], case["page"], case["ctx"]
        shared, per = c // page, -(-(c + T) // page)              # the prompt's whole pages are shared
        n_pages = shared + B * (per - shared)
        order, tab = r.permutation(n_pages), np.zeros((B, per), np.int32)
        for b in range(B):
            tab[b, :shared] = order[:shared]
            tab[b, shared:] = order[shared + b * (per - shared):shared + (b + 1) * (per - shared)]
        k = torch.randint(-(1 << 20), 1 << 20, (n_pages, nl, nkv, page, hd), generator=g, device=dev, dtype=torch.int32)
        v = torch.randint(-(1 << 20), 1 << 20, (n_pages, nl, nkv, page, hd), generator=g, device=dev, dtype=torch.int32)
        s |= {"k": k, "v": v, "table": torch.from_numpy(tab).to(dev), "ctx": ints([c] * B),
              "path0": ints([b * case["accept"] for b in range(B + 1)]),
              "path": ints(sum((_path(r, T, case["accept"]) for _ in range(B)), []))}
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    return {"attention": _attention, "logprobs": _logprobs, "compact": _compact}[s["op"]](s)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _attention(s):
    nh, nkv, hd, _ = SHAPES[s["shape"]]
    if own:
        _library().tree_attn(_pages(s), 0, s["seqs"], s["ctx"].data_ptr(), s["row0"].data_ptr(), s["parent"].data_ptr(), s["seqs"] * s["nodes"],
                             s["max_ctx"], s["q"].data_ptr(), nh, s["window"], s["out"].data_ptr(), _stream())
        return s["out"]
    B, T, G, dev = s["seqs"], s["nodes"], nh // nkv, s["q"].device
    L = s["max_ctx"] + T
    # each sequence's cache in the order of its positions: [B, KV heads, L, head width]
    at = torch.arange(L, device=dev)
    page = s["table"].long()[:, (at // s["page"]).clamp(max=s["table"].shape[1] - 1)]
    k = s["k"][page, 0, :, at % s["page"]].double().permute(0, 2, 1, 3)
    v = s["v"][page, 0, :, at % s["page"]].double().permute(0, 2, 1, 3)
    # ancestors: the closure of the parent relation (64 nodes at most: six squarings)
    parent = s["parent"].view(B, T, 1).long()
    a = (torch.arange(T, device=dev) == parent).float() + torch.eye(T, device=dev)
    a = a @ a
    a = (a @ a).clamp(max=1.0)
    a = (a @ a).clamp(max=1.0)
    a = (a @ a).clamp(max=1.0)
    a = (a @ a).clamp(max=1.0)
    a = (a @ a).clamp(max=1.0)
    sees = a > 0                                                   # [B, node, ancestor or itself]
    depth = sees.sum(2) - 1
    ctx = s["ctx"].long().view(B, 1, 1)
    place = at.view(1, 1, L)
    slot = (place - ctx).clamp(0, T - 1)
    in_tree = (place >= ctx) & (place < ctx + T) & sees.gather(2, slot.expand(B, T, L))
    # a slot's position in its sequence: a context position is its own, a node's is its depth's
    where = torch.where(place < ctx, place, ctx + depth.unsqueeze(1).gather(2, slot))
    ok = (place < ctx) | in_tree
    if s["window"] >= 0:
        ok = ok & (where > ctx + depth.unsqueeze(2) - s["window"])
    ok = ok.view(B, 1, T, 1, L)
    q = s["q"].view(B, T, nkv, G, hd).double().permute(0, 2, 1, 3, 4).reshape(B, nkv, T * G, hd)
    z = ((q @ k.transpose(2, 3)) * 2.0 ** -32).float() * torch.tensor(1.0 / math.sqrt(hd), dtype=torch.float32, device=dev)
    z = z.mul_(16384.0)
    zi = torch.copysign((z.abs().double() + 0.5).floor_(), z.double()).to(torch.int64)
    zi = zi.view(B, nkv, T, G, L)
    top = torch.where(ok, zi, -(1 << 40)).amax(4, keepdim=True)
    far = (top - zi).clamp_(0, FAR)
    g = (far * LOG2E + 16383) >> 14
    n, f = g >> 30, g & (ONE - 1)
    x = ONE - f
    p = ((EXP2[6] * x) >> 30) + EXP2[5]
    p = ((p * x) >> 30) + EXP2[4]
    p = ((p * x) >> 30) + EXP2[3]
    p = ((p * x) >> 30) + EXP2[2]
    p = ((p * x) >> 30) + EXP2[1]
    p = ((p * x) >> 30) + EXP2[0]
    e = torch.where(f > 0, p >> (n + 1).clamp(max=62), ONE >> n.clamp(max=62))
    e = torch.where(ok & (n < 32), e, 0).double().view(B, nkv, T * G, L)
    o = (e @ v) / e.sum(3, keepdim=True) * 2.0 ** -16
    return o.float().view(B, nkv, T, G, hd).permute(0, 2, 1, 3, 4).reshape(B * T, nh * hd)


def _logprobs(s):
    n, v, top = s["rows"], s["vocab"], s["top"]
    if own:
        _library().logprobs(s["x"].data_ptr(), n, v, v + s["pad"], s["row"].data_ptr(), s["tok"].data_ptr(), s["row"].numel(),
                            s["logprob"].data_ptr(), s["lse"].data_ptr(), s["entropy"].data_ptr(), top, s["ids"].data_ptr() if top else None,
                            s["best"].data_ptr() if top else None, _stream())
        return [s["logprob"], s["lse"], s["entropy"]] + ([s["ids"], s["best"]] if top else [])
    x = s["x"][:, :v]
    m = x.amax(1, keepdim=True)
    d = x - m
    e = d.exp()
    t = e.sum(1)
    lse = m[:, 0] + t.log()
    entropy = t.log() - torch.where(e > 0, e * d, 0.0).sum(1) / t
    logprob = x[s["row"].long(), s["tok"].long()] - lse[s["row"].long()]
    if not top:
        return [logprob, lse, entropy]
    # order by value, equal ones lowest id first: one whole-number key for each entry
    b = (x + 0.0).view(torch.int32).long()
    key = torch.where(b < 0, b ^ 0x7FFFFFFF, b) * (1 << 32) + ((1 << 32) - 1 - torch.arange(v, device=x.device))
    ids = ((1 << 32) - 1) - (key.topk(top, 1).values & ((1 << 32) - 1))
    return [logprob, lse, entropy, ids.int(), x.gather(1, ids) - lse.unsqueeze(1)]


def _compact(s):
    if own:
        _library().kv_compact(_pages(s), s["seqs"], s["ctx"].data_ptr(), s["path0"].data_ptr(), s["path"].data_ptr(),
                              s["seqs"] * s["accept"], _stream())
        return [s["k"], s["v"]]
    B, A, page = s["seqs"], s["accept"], s["page"]
    src = s["ctx"].long().view(B, 1) + s["path"].long().view(B, A)
    dst = s["ctx"].long().view(B, 1) + torch.arange(A, device=src.device)
    table = s["table"].long()
    sp, dp = table.gather(1, src // page), table.gather(1, dst // page)
    for c in (s["k"], s["v"]):
        c[dp, :, :, dst % page] = c[sp, :, :, src % page]
    return [s["k"], s["v"]]


# ------------------------------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    if case["op"] == "compact":
        return None                                                # rows are moved, none is computed
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        n, v, top = s["rows"], s["vocab"], s["top"]
        lse, entropy, ids, best, step = [], [], [], [], max(1, 16_000_000 // v)
        for r0 in range(0, n, step):
            x = s["x"][r0:r0 + step, :v].double()
            lg = torch.logsumexp(x, 1)
            p = (x - lg.unsqueeze(1)).exp()
            lse.append(lg)
            entropy.append(-torch.special.xlogy(p, p).sum(1))
            if top:
                val, at = torch.sort(x, dim=1, descending=True, stable=True)
                ids.append(at[:, :top])
                best.append(val[:, :top] - lg.unsqueeze(1))
        lse = torch.cat(lse)
        row = s["row"].long()
        logprob = s["x"].double()[row, s["tok"].long()] - lse[row] if n * v < 1 << 26 else s["x"][row, s["tok"].long()].double() - lse[row]
        got = [logprob, lse, torch.cat(entropy)]
        return got + [torch.cat(ids), torch.cat(best)] if top else got
    nh, nkv, hd, _ = SHAPES[case["shape"]]
    B, T, G, page, w = s["seqs"], s["nodes"], nh // nkv, s["page"], s["window"]
    out = torch.zeros(B * T, nkv, G, hd, dtype=torch.float64, device=s["q"].device)
    table, ctxs, parents = s["table"].tolist(), s["ctx"].tolist(), s["parent"].view(B, T).tolist()
    for b in range(B):
        c = ctxs[b]
        rows = [(table[b][j // page], j % page) for j in range(c + T)]
        pg, off = (torch.tensor(x, device=out.device) for x in zip(*rows))
        kk, vv = s["k"][pg, 0, :, off].double(), s["v"][pg, 0, :, off].double()      # [L, KV heads, width]
        chains = []
        for i in range(T):
            chain = [i]
            while parents[b][chain[-1]] >= 0:
                chain.append(parents[b][chain[-1]])
            chains.append(chain[::-1])
        for i, chain in enumerate(chains):
            p = c + len(chain) - 1
            first = 0 if w < 0 else max(0, p - w + 1)
            # the ancestor at depth t stands at position c + t
            see = list(range(min(first, c), c)) + [c + a for t, a in enumerate(chain) if c + t >= first]
            at = torch.tensor(see, device=out.device)
            q = s["q"][b * T + i].view(nkv, G, hd).double()
            score = torch.einsum("gad,lgd->gal", q, kk[at])         # whole numbers below 2^53
            z = (score / 4294967296.0).float() * np.float32(1.0 / math.sqrt(hd))
            z = z.double() * 16384.0
            grid = torch.where(z < 0, torch.ceil(z - 0.5), torch.floor(z + 0.5)) / 16384.0
            e = torch.exp(grid - grid.amax(2, keepdim=True))
            out[b * T + i] = torch.einsum("gal,lgd->gad", e, vv[at]) / e.sum(2, keepdim=True) / 65536.0
    return out.view(B * T, nh * hd)
