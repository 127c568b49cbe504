"""Drafted trees and scored prompts on tensor-parallel models: a group of one rank on one GPU, larger ones
on boxes that have the GPUs."""
import os
import socket

import numpy as np
import pytest

import spb200
import spmodel
from test_gpu_tp import MODELS, _n_gpus

pytestmark = pytest.mark.gpu


def _tree_results(m, cfg):
    """a scored prompt, two tree steps with their commits, and the steps that follow"""
    r = np.random.default_rng(9)
    s = m.session(96)
    out = {}
    def keep(name, res):
        for f in ("logits", "argmax", "logprob", "entropy", "top_id", "top_logprob"):
            out[f"{name}_{f}"] = getattr(res, f)
    keep("score", s.score(spmodel.gen_tokens(52, 37, cfg.n_vocab), top=4, logits=True))
    for i, (parent, path) in enumerate((([-1, 0, 0, 1, 2, -1, 4], [0, 2, 4]), ([-1, -1, 1], [1]))):
        keep(f"tree{i}", s.tree_step(r.integers(0, cfg.n_vocab, len(parent)), parent, top=3))
        s.tree_commit(path)
        out[f"step{i}"] = s.step(int(r.integers(0, cfg.n_vocab))).copy()
    out["position"] = np.array(s.position())
    s.close()
    return out


def _tree_rank(rank, world, port, out_dir, name):
    import torch.distributed as dist
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world)
    tp = spb200.TensorParallel(spb200.tp_uid_from_dist(), rank, world, device=rank)
    m = spb200.Model.synthetic_tp(MODELS[name], tp, seed=3)
    res = _tree_results(m, MODELS[name])
    m.free()
    tp.close()
    dist.destroy_process_group()
    np.savez(os.path.join(out_dir, f"rank{rank}.npz"), **res)


@pytest.mark.parametrize("world,name", [(1, "micro_gemma"), (1, "micro_qwen"), (2, "micro_gemma"), (2, "micro_qwen"), (8, "gemma12b_w2")])
def test_tp_trees_and_scores_match_single_gpu(cuda_ok, tmp_path, world, name):
    """Drafted trees, their commits and scored prompts on every rank: the whole model's bytes."""
    if _n_gpus() < world:
        pytest.skip(f"needs {world} GPUs")
    import torch.multiprocessing as mp
    with socket.socket() as sk:
        sk.bind(("127.0.0.1", 0))
        port = sk.getsockname()[1]
    mp.spawn(_tree_rank, args=(world, port, str(tmp_path), name), nprocs=world, join=True)
    m = spb200.Model.synthetic(MODELS[name], seed=3)
    want = _tree_results(m, MODELS[name])
    m.free()
    for r in range(world):
        got = np.load(tmp_path / f"rank{r}.npz")
        for k, w in want.items():
            assert np.array_equal(np.ascontiguousarray(got[k]).view(np.uint8), np.ascontiguousarray(w).view(np.uint8)), f"rank {r} {k}"
