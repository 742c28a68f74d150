"""Paged 8-bit cache, beam search and GPT's answers on CPU tensors at the borders of what their calls allow."""
import pytest
import torch

from noeira_b200.models.gpt import GPT
from noeira_b200.ops import beam, kvcache

I32 = torch.int32


def ints(v):
    return torch.tensor(v, dtype=I32)


# ------------------------------------------------------------------------------------------------ plan
@pytest.mark.parametrize("block", [16, 32])
def test_rows_hold_max_len_tokens_and_no_more(block):
    c = kvcache.PagedKVCache(1, 1, 64, 8, 2, 18, block, device="cpu")
    p = c.plan(ints([18, 17]), 35)
    assert p.positions.tolist() == list(range(18)) + list(range(17)) and min(p.slots.tolist()) >= 0
    assert c.plan(ints([0, 1]), 1).positions.tolist() == [17]
    for new in ([1, 0], [0, 10]):
        with pytest.raises(RuntimeError, match="no room"):
            c.plan(ints(new), sum(new))
    assert c.lengths.tolist() == [18, 18]


def test_plan_tokens_takes_a_limit():
    ok = dict(tables=torch.full((2, 3), -1, dtype=I32), lengths=ints([0, 0]), new_lens=ints([20, 1]), free=ints([0, 1, 2, 3]), free_count=ints([4]), block=16, tokens=21)
    kvcache.plan_tokens(**{**ok, "free_count": ints([4]), "max_len": 20})
    kvcache.plan_tokens(**{**ok, "free_count": ints([4]), "max_len": 1 << 40})        # no more than the table has room for
    with pytest.raises(RuntimeError, match=r"rows \[0\]"):
        kvcache.plan_tokens(**ok, max_len=19)
    with pytest.raises(ValueError, match="max_len"):
        kvcache.plan_tokens(**ok, max_len=-1)


@pytest.mark.parametrize("bad", [8, 1 << 27, 1 << 28, -1])
@pytest.mark.parametrize("place", ["table", "stack"])
def test_plan_names_blocks_that_are_none(bad, place):
    c = kvcache.PagedKVCache(1, 1, 64, 8, 2, 64, 16, device="cpu")
    c.plan(ints([5, 5]), 10)
    if place == "table":
        c.tables[0, 0] = bad
    else:
        c.free[int(c.free_count) - 1] = bad
    with pytest.raises(ValueError, match=r"rows \[0\]"):
        c.plan(ints([13, 3]), 16)
    for blocks in (0, (1 << 27) + 1):
        with pytest.raises(ValueError, match="blocks"):
            kvcache.plan_tokens(c.tables, c.lengths, ints([1, 1]), c.free, c.free_count, 16, 2, blocks=blocks)


def test_a_plan_that_raises_changes_nothing():
    """Blocks that a refused plan wrote into tables were neither free nor a row's after a reset of other rows."""
    c = kvcache.PagedKVCache(1, 1, 64, 3, 2, 64, 16, device="cpu")
    c.plan(ints([16, 0]), 16)
    before = [t.clone() for t in (c.tables, c.lengths, c.free, c.free_count)]
    with pytest.raises(RuntimeError, match=r"rows \[1\]"):
        c.plan(ints([20, 33]), 53)
    c.free[0] = 3                                             # no block of the cache
    before[2][0] = 3
    with pytest.raises(ValueError, match=r"rows \[1\]"):
        c.plan(ints([1, 1]), 2)
    assert all(torch.equal(a, b) for a, b in zip(before, (c.tables, c.lengths, c.free, c.free_count)))
    c.reset([1])
    assert int(c.free_count) == 2
    c.plan(ints([0, 32]), 32)


def test_reorder_leaves_the_caches_tensors_in_their_place():
    """A captured step holds the addresses of tables, lengths and spare blocks."""
    c = kvcache.PagedKVCache(1, 1, 64, 12, 3, 40, 16, device="cpu", spares=True)
    c.plan(ints([20, 0, 0]), 20)
    held = c.tables, c.lengths, c.spare
    at = [t.data_ptr() for t in held]
    c.reorder(ints([[0, 0, 0]]))
    assert [t.data_ptr() for t in (c.tables, c.lengths, c.spare)] == at
    assert held[1].tolist() == [20] * 3 and held[0][:, 0].unique().numel() == 1 and held[0][:, 1].unique().numel() == 3
    assert held[2][1:].tolist() == [-1, -1]
    c.refill_spares()
    assert int(held[2].min()) >= 0 and held[2].unique().numel() == 3


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("tokens", [1, 20, 60])
def test_attention_nan_in_the_cache_reaches_only_who_sees_it(tokens):
    import kv_cases as C
    d = C.attention_inputs(([50, 10], [tokens, tokens], 4, 2, 64, 16))
    q, rest = d["q"][: d["T"], 1:5], (d["scale"], d["tables"], d["starts"], d["ends"])
    want = kvcache.paged_attention(q, d["codes"], *rest)
    raw = d["codes"].view(torch.uint8)
    raw[1, d["tables"][1, 0], 1, 12, 5] = 0x7F                # a value: row 1, place 12, head 1, dimension 5
    raw[0, d["tables"][0, 3], 0, 4, 9] = 0xFF                 # a key: row 0, place 52, head 0
    got = kvcache.paged_attention(q, d["codes"], *rest)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[tokens + 2:, 2:, 5] = True
    bad[2: tokens, :2] = True
    assert torch.equal(torch.isnan(got), bad) and torch.equal(got[~bad], want[~bad])


# ------------------------------------------------------------------------------------------------ beams
def test_select_refuses_vocabularies_whose_last_part_passes_32_bits():
    for vocab in (0x7fff0001, 0x7ffffeff):                    # no memory behind it: the sizes alone decide
        with pytest.raises(ValueError, match="tokens"):
            beam.beam_select(torch.empty(1, 1, vocab, dtype=torch.bfloat16, device="meta"), torch.empty(1, 1, device="meta"))


# ------------------------------------------------------------------------------------------------ GPT
def small(**kw):
    return GPT(**{**dict(vocab=32, seq=20, dim=64, layers=1, heads=1, seed=3), **kw}).eval()


def test_gpt_answers_up_to_its_last_position():
    """``seq`` is no multiple of the block."""
    m = small()
    cache = m.new_cache(1, 20)
    ids = torch.arange(19)
    m.forward_cached(ids, cache, cache.plan(ints([19]), 19))
    assert bool(torch.isfinite(m.forward_cached(ids[:1], cache, cache.plan(ints([1]), 1))).all())
    with pytest.raises(RuntimeError, match="no room"):
        cache.plan(ints([1]), 1)
    assert len(m.generate([[1] * 15], max_new=5)[0]) == 5


def test_gpt_refuses_a_cache_of_longer_rows():
    m = small()
    cache = kvcache.PagedKVCache(1, 1, 64, 4, 1, 21, device="cpu")
    plan = cache.plan(ints([2]), 2)
    with pytest.raises(ValueError, match="20 positions"):
        m.forward_cached(torch.zeros(2, dtype=torch.int64), cache, plan)


def test_gpt_looks_up_places_inside_its_tables_only():
    """What a refused plan holds on the GPU, where nothing raises: rows that start behind the tokens, places of any size."""
    m = small()
    cache = m.new_cache(3, 20)
    plan = cache.plan(ints([2, 3, 0]), 5)
    ids = torch.tensor([1, 2, 3, 4, 5])
    want = m.forward_cached(ids, cache, plan)
    got = m.forward_cached(ids, cache, plan._replace(starts=ints([0, 2, 5, 9])))
    assert torch.equal(got[:2], want[:2]) and bool(torch.isfinite(got).all())
    got = m.forward_cached(ids, cache, plan._replace(positions=ints([0, 1, 20, -7, 0x7fffffff])))
    assert torch.equal(got[0], want[0]) and bool(torch.isfinite(got).all())


def test_gpt_refuses_ids_that_are_not_the_plans():
    m = small()
    cache = m.new_cache(2, 20)
    plan = cache.plan(ints([2, 1]), 3)
    for ids in (torch.zeros(1, dtype=torch.int64), torch.zeros(4, dtype=torch.int64), torch.zeros(1, 3, dtype=torch.int64)):
        with pytest.raises(ValueError, match="3 tokens"):
            m.forward_cached(ids, cache, plan)
    with pytest.raises(ValueError, match="one at least"):
        m.forward_cached(torch.zeros(0, dtype=torch.int64), cache, cache.plan(ints([0, 0]), 0))


@pytest.mark.parametrize("bad", [32, -1, 1 << 40])
def test_gpt_refuses_prompts_of_other_tokens(bad):
    m = small()
    for answer in (m.beam_search, m.generate):
        with pytest.raises(ValueError, match="32 tokens"):
            answer([[1, 2], [3, bad, 4]], max_new=2)
    assert len(m.generate([[0, 31]], max_new=2)[0]) == 2


def gradients(m, ids, between):
    m.zero_grad()
    logits = m.forward(ids)
    between()
    m.vjp(torch.cos(torch.arange(logits.numel(), device=logits.device).reshape(logits.shape)).to(logits.dtype))
    return {k: p.grad.clone() for k, p in m.named_params()}


@pytest.mark.parametrize("tie", [False, True])
def test_answers_between_forward_and_vjp_change_no_gradient(tie):
    m = small(tie=tie)
    ids = torch.randint(0, 32, (2, 20), generator=torch.Generator().manual_seed(1))
    want = gradients(m, ids, lambda: None)
    cache = m.new_cache(1, 20)

    def steps():
        plan = cache.plan(ints([3]), 3)
        m.forward_cached(torch.tensor([1, 2, 3]), cache, plan)

    for between in (lambda: m.generate([[1, 2, 3], [4]], max_new=4), lambda: m.beam_search([[5, 6]], beams=3, max_new=4), steps):
        got = gradients(m, ids, between)
        assert all(torch.equal(got[k], want[k]) for k in want)
    with pytest.raises(ValueError):                           # a call that fails on its way leaves no trace either
        m.generate([[1, 2, 3]], max_new=4, eos=32)
    logits = m.forward(ids)
    with pytest.raises(ValueError):
        m.generate([[1, 2, 3]], max_new=4, eos=32)
    m.zero_grad()
    m.vjp(torch.cos(torch.arange(logits.numel()).reshape(logits.shape)).to(logits.dtype))
    assert all(torch.equal(p.grad, want[k]) for k, p in m.named_params())


def test_saved_kept_reaches_parts_without_parameters():
    from noeira_b200 import nn
    b = nn.TransformerBlock(64, 1, 64, norm="rms", ffn="swiglu", mask="causal")
    x = torch.randn(1, 5, 64)
    b.forward(x)
    before = [dict(vars(m)) for m in (*b.modules(), b.ffn.act)]
    with b.saved_kept():
        b.forward(torch.randn(2, 3, 64))
        b.late = 1
    for m, held in zip((*b.modules(), b.ffn.act), before):
        assert vars(m).keys() == held.keys() and all(vars(m)[k] is held[k] for k in held)


def test_block_with_grouped_heads():
    """Prompts in pieces and single tokens.  Sums in fp32, and codes that a growing scale moved below 2^-6 once more: see the
    logits' test, of which this is one layer."""
    import gpt_serving as G
    for got, want in zip(*G.attention_block("cpu")):
        assert float((got - want).abs().max()) <= 1e-4 * float(want.abs().max())
