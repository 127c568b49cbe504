"""How a call of the log probabilities is cut, without a GPU."""
import os
import subprocess

import spb200


PLAN = r"""
#include <cstdio>
#include <cstdlib>
#include "spb_logprob_plan.h"
int main(int n, char **v) {   // rows, vocab, largest cluster, largest cluster with unused memory
  const int most = atoi(v[3]), padded = atoi(v[4]);
  const auto p = spb::plan_logprobs(atoi(v[1]), atoi(v[2]), [&](int c, int pad) { return c <= (pad ? padded : most); });
  printf("%d %d %d %d\n", p.parts, p.per, p.ctas, p.pad);
}
"""


def test_logprob_clusters_that_do_not_fit(tmp_path):
    """A device that runs smaller clusters than a call wants gets smaller ones, and the same parts of a row."""
    (tmp_path / "plan.cc").write_text(PLAN)
    csrc = os.path.join(os.path.dirname(os.path.abspath(spb200.__file__)), "csrc")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", csrc, "-o", tmp_path / "plan", tmp_path / "plan.cc"], check=True)
    for rows, vocab in ((1, 1), (1, 16385), (1, 262144), (1, 1 << 22), (3, 100000), (64, 262144), (150, 151936), (1000, 151936), (1 << 26, 1 << 22)):
        plans = {}
        for most, padded in ((16, 16), (16, 8), (8, 8), (8, 0), (5, 3), (2, 1), (1, 1)):
            out = subprocess.run([tmp_path / "plan", *map(str, (rows, vocab, most, padded))], check=True, capture_output=True, text=True)
            parts, per, ctas, pad = plans[most, padded] = tuple(map(int, out.stdout.split()))
            assert 1 <= ctas <= (max(1, padded) if pad and ctas > 1 else most) and pad in (0, 52 * 1024, 92 * 1024)
            assert (parts, per) == plans[16, 16][:2] and ctas <= plans[16, 16][2]
            assert (parts - 1) * per < vocab <= parts * per and per % 4 == 0 and parts <= 16
            assert (ctas - 1) * -(-parts // ctas) < parts         # every CTA has a part
        if plans[16, 16][2] > 5:
            assert plans[8, 0][2] > 2 and plans[8, 0][3] == 0 and plans[1, 1][2] == 1


def test_tokens_times_rows_are_limited():
    """With tok_row every row looks through the list: a call that would take minutes is refused; without, none is."""
    def call(rows, n_tok, tok_row=256):
        try:
            spb200.logprobs(256, rows, 8, 8, tok_row, 256, n_tok, 256, None, None, 0, None, None)
        except spb200.SpbError as e:
            return e.code
    for rows, n_tok in ((1 << 26, 1 << 26), ((1 << 20) + 1, 1 << 20), (1 << 26, (1 << 14) + 1)):
        assert call(rows, n_tok) == spb200.SPB_EUNSUPPORTED
    for rows, n_tok, tok_row in ((1 << 20, 1 << 20, 256), (1 << 26, 1 << 14, 256), (1 << 26, 1 << 26, None)):
        assert call(rows, n_tok, tok_row) == spb200.SPB_EBADARG      # (only its pointers are bad)
