"""GPT answering prompts over the paged 8-bit cache, on CPU tensors in fp32."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import gpt_serving as G

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("tie", [False, True])
def test_logits_equal_a_forward_over_quantised_keys_and_values(tie):
    """Prompts and single tokens, against the whole sequence at once with keys and values rounded block by block.  A scale that
    grows within a block moves earlier codes below 2^-6 of it once more: 2^-10 / 448 of the block's largest value, 2.2e-6; sums in
    fp32 of the same order.  Both pass two layers: 1e-4 of the logits' size covers forty such errors in each of them."""
    m = G.model("cpu", tie)
    prompts, steps = G.sequences()
    got = G.cached_logits(m, prompts, steps)
    for r, (p, s) in enumerate(zip(prompts, steps)):
        want = G.quantised_logits(m, p + s, block=16)
        for n in range(len(s) + 1):
            w = want[len(p) - 1 + n]
            assert float((got[r][n] - w).abs().max()) <= 1e-4 * float(w.abs().max()), (r, n)


def test_prompt_in_pieces_gives_the_same_logits():
    m = G.model("cpu")
    p = list(range(40))
    whole = G.cached_logits(m, [p], [[]])[0][0]
    cache = m.new_cache(1, 64)
    for piece in (p[:7], p[7:16], p[16:39], p[39:]):
        plan = cache.plan(torch.tensor([len(piece)], dtype=torch.int32), len(piece))
        last = m.forward_cached(torch.tensor(piece), cache, plan)
    assert float((whole - last[0]).abs().max()) <= 1e-4 * float(whole.abs().max())


def test_beam_search_is_what_its_steps_say():
    """Scores are the summed log-probabilities of the sequences under the same quantised model, best first, all different."""
    m = G.model("cpu")
    prompts = [[3, 1, 4, 1, 5, 9, 2, 6], list(range(16)), [7]]
    seqs, scores = m.beam_search(prompts, beams=4, max_new=21)
    for r, p in enumerate(prompts):
        assert len({tuple(s) for s in seqs[r]}) == 4 and torch.equal(scores[r].sort(descending=True).values, scores[r])
        for j in range(4):
            lp = torch.log_softmax(G.quantised_logits(m, p + seqs[r][j], block=16), -1)
            total = sum(float(lp[len(p) - 1 + n, t]) for n, t in enumerate(seqs[r][j]))
            # 21 log-probabilities of logits that are 1e-4 of their size off, at most twice each
            assert abs(total - float(scores[r, j])) <= 21 * 2e-4 * float(lp.abs().max())
    assert m.generate(prompts, max_new=9) == [s[0] for s in m.beam_search(prompts, beams=1, max_new=9)[0]]


def test_beam_search_stops_at_eos():
    m = G.model("cpu")
    eos = m.generate([[3, 1, 4]], max_new=5)[0][2]
    out = m.generate([[3, 1, 4], [2]], max_new=30, eos=eos)
    assert out[0][-1] == eos and eos not in out[0][:-1]
    seqs, _ = m.beam_search([[3, 1, 4]], beams=3, max_new=30, eos=eos)
    assert all(eos not in s[:-1] for s in seqs[0])


def test_refusals():
    from noeira_b200 import nn
    m = G.model("cpu")
    for kw in (dict(prompts=[]), dict(prompts=[[]]), dict(prompts=[[1]], beams=0), dict(prompts=[[1]], max_new=0), dict(prompts=[[1]], max_new=m.seq), dict(prompts=[[1]], beams=33)):
        with pytest.raises(ValueError):
            m.beam_search(**{**dict(beams=2, max_new=4), **kw})
    cache = m.new_cache(1, 8)
    plan = cache.plan(torch.tensor([2], dtype=torch.int32), 2)
    for blk in (nn.SelfAttention(128, 2), nn.SelfAttention(128, 2, mask="causal", rope_theta=1e4)):
        with pytest.raises(ValueError, match="causal"):
            blk.forward_cached(torch.zeros(2, 128), cache, 0, plan)
    with pytest.raises(RuntimeError, match="no room"):
        cache.plan(torch.tensor([15], dtype=torch.int32), 15)


def test_example_answers(tmp_path):
    (tmp_path / "corpus.txt").write_text("the quick brown fox jumps over the lazy dog. " * 40)
    r = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "gpt_char.py"), str(tmp_path / "corpus.txt"), "--steps", "2", "--seq", "32", "--batch", "2",
                        "--answer", "the q", "--tokens", "6", "--beams", "2"], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    assert len([l for l in r.stdout.splitlines() if "'the q" in l]) == 2
