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
