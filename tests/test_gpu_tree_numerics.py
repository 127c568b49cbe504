"""Values at which the kernels that verify drafted trees can go wrong: every distance of a score below
its maximum."""
import numpy as np
import pytest
import torch

import spb200
from test_gpu_tree import dev, errs, exp_fixed, u32

pytestmark = pytest.mark.gpu

ONE = 1 << 30


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
