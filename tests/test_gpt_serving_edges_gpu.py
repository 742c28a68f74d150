"""GPT's answers on the GPU at the borders of what its calls allow."""
import pytest
import torch

import gpt_serving as G

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def reported(match):
    from noeira_b200.ops import check_status
    from noeira_b200.ops.status import DeviceStatusError
    with pytest.raises(DeviceStatusError, match=match):
        check_status()


@pytest.mark.parametrize("new,tokens", [([10, 10, 10], 25), ([10, 10, 60], 80)])
def test_rows_beside_a_refused_one_get_their_logits(new, tokens):
    """The third row outgrows the token dimension, or the model's positions; the first two are answered as if it were not there."""
    from noeira_b200.ops import check_status
    m = G.model("cuda")
    ids = torch.randint(0, 64, (tokens,), generator=torch.Generator().manual_seed(4)).cuda()
    cache = m.new_cache(3, 50)
    want = m.forward_cached(ids[:20], cache, cache.plan(ints([10, 10, 0]), 20), max_new=10)
    check_status()
    cache = m.new_cache(3, 50)
    got = m.forward_cached(ids, cache, cache.plan(ints(new), tokens), max_new=60)
    reported("no room")
    assert cache.lengths.tolist() == [10, 10, 0] and bool(torch.isfinite(got).all())
    # other launches for another number of tokens: both round to bf16 (2^-8) in two layers
    assert float((got[:2].float() - want[:2].float()).norm()) <= 2 * 2 * 3 * 2.0 ** -8 * float(want[:2].float().norm())


@pytest.mark.parametrize("tie", [False, True])
def test_answers_between_forward_and_vjp_change_no_gradient(tie):
    m = G.model("cuda", tie)
    ids = torch.randint(0, 64, (2, 64), generator=torch.Generator().manual_seed(1)).cuda()
    g = (torch.cos(torch.arange(2 * 64 * 64, device="cuda")) / 64).reshape(2, 64, 64).bfloat16()
    got = []
    for between in (lambda: None, lambda: None, lambda: m.generate([[1, 2, 3], [4]], max_new=4), lambda: m.beam_search([[5, 6]], beams=3, max_new=4)):
        m.zero_grad()
        m.forward(ids)
        between()
        m.vjp(g)
        got.append({k: p.grad.clone() for k, p in m.named_params()})
    # the embedding's rows are summed by atomics in no fixed order: fp32 sums of up to 128 terms, whose order moves a sum of
    # magnitude A by 128 * 2^-24 A; all else repeats bit by bit
    for other in got[1:]:
        for k, w in got[0].items():
            if torch.equal(other[k], w):
                continue
            assert "wte" in k or "wpe" in k, k
            assert float((other[k] - w).abs().max()) <= 2 * 128 * 2.0 ** -24 * 128 * float(w.abs().max()), k


def test_block_with_grouped_heads():
    """Attention's output and its weights round by 2^-8 each, the projection's output once more, and a flipped code doubles it."""
    for got, want in zip(*G.attention_block("cuda")):
        assert float((got - want).norm()) <= 2 * 3 * 2.0 ** -8 * float(want.norm())
