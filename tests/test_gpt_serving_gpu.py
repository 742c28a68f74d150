"""GPT answering prompts over the paged 8-bit cache on the GPU."""
import pytest
import torch

import gpt_serving as G

pytestmark = pytest.mark.gpu

# Against the same layers over a whole sequence, with keys and values rounded and attention in 64 bits: the outputs of attention
# differ by their rounding and that of the weights (2^-8 each, of values of one size), and each of two layers adds as much again
# to what the residual stream carries in bf16 (2^-8): 2 * 3 * 2^-8 of the logits' size, and a factor of two for a flipped code.
TOLERANCE = 2 * 2 * 3 * 2.0 ** -8


@pytest.mark.parametrize("tie", [False, True])
def test_logits(tie):
    from noeira_b200.ops import check_status
    m = G.model("cuda", tie)
    prompts, steps = G.sequences()
    got = G.cached_logits(m, prompts, steps)
    check_status()
    for r, (p, s) in enumerate(zip(prompts, steps)):
        want = G.quantised_logits(m, p + s, block=16)
        for n in range(len(s) + 1):
            w = want[len(p) - 1 + n]
            assert float((got[r][n] - w).norm()) <= TOLERANCE * float(w.norm()), (r, n)


def test_beam_search():
    m = G.model("cuda")
    prompts = [[3, 1, 4, 1, 5, 9, 2, 6], list(range(16)), [7]]
    seqs, scores = m.beam_search(prompts, beams=4, max_new=21)
    scores = scores.cpu()
    for r, p in enumerate(prompts):
        assert len({tuple(s) for s in seqs[r]}) == 4 and torch.equal(scores[r].sort(descending=True).values, scores[r])
        for j in range(4):
            x = G.quantised_logits(m, p + seqs[r][j], block=16).double()
            lp = torch.log_softmax(x, -1)
            total = sum(float(lp[len(p) - 1 + n, t]) for n, t in enumerate(seqs[r][j]))
            # a log-probability moves by at most twice the largest error of a logit
            assert abs(total - float(scores[r, j])) <= 21 * 2 * TOLERANCE * float(x.abs().max())
    assert m.generate(prompts, max_new=9) == [s[0] for s in m.beam_search(prompts, beams=1, max_new=9)[0]]


def test_cache_too_small_is_reported():
    from noeira_b200.ops import check_status
    from noeira_b200.ops.status import DeviceStatusError
    m = G.model("cuda")
    cache = m.new_cache(2, 64, blocks=3)
    cache.plan(torch.tensor([20, 40], dtype=torch.int32, device="cuda"), 60)
    with pytest.raises(DeviceStatusError, match="no room"):
        check_status()


def test_decode_steps_in_a_captured_graph():
    """A decode step with its plan, captured once and replayed, writes the cache and gives the logits of eager steps."""
    from noeira_b200.ops import check_status
    m = G.model("cuda")
    prompts, steps = G.sequences()
    want = G.cached_logits(m, prompts, steps)
    rows = len(prompts)
    cache = m.new_cache(rows, 64)
    one = torch.ones(rows, dtype=torch.int32, device="cuda")
    ids = torch.zeros(rows, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):                    # once before the capture, on the stream that captures: lazy workspaces
        warm = m.new_cache(rows, 64)
        m.forward_cached(ids, warm, warm.plan(one, rows), max_new=1)
    side.synchronize()
    first = torch.tensor([t for p in prompts for t in p], device="cuda")
    plan = cache.plan(torch.tensor([len(p) for p in prompts], dtype=torch.int32, device="cuda"), first.numel())
    m.forward_cached(first, cache, plan, max_new=max(len(p) for p in prompts))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        logits = m.forward_cached(ids, cache, cache.plan(one, rows), max_new=1)
    for n in range(len(steps[0])):
        ids.copy_(torch.tensor([s[n] for s in steps]))
        g.replay()
        for r in range(rows):
            assert torch.equal(logits[r].float().cpu(), want[r][n + 1]), (n, r)
    check_status()
