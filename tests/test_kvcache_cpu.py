"""Paged 8-bit cache and beam search on CPU tensors, against definitions in 64 bits, and every refusal."""
import math

import numpy as np
import pytest
import torch

import kv_cases as C
import kv_oracle as O
from noeira_b200.ops import beam, kvcache

I32 = torch.int32


def ints(v):
    return torch.tensor(v, dtype=I32)


@pytest.mark.parametrize("lengths,new,block,spare,pad", C.PLANS)
def test_plan(lengths, new, block, spare, pad):
    tables, blocks, left = C.paged(lengths, block, 3, spare_blocks=sum(-(-n // block) + 1 for n in new) + spare, extra_width=-(-max(new) // block) + 1)
    free, count = ints(left.tolist()), ints([len(left)])
    tokens = sum(new) + pad
    want, refused = O.plan(tables, lengths, new, left, len(left), block, tokens)
    assert not refused
    t = torch.from_numpy(tables.copy())
    p = kvcache.plan_tokens(t, ints(lengths), ints(new), free, count, block, tokens)
    got = dict(tables=t, starts=p.starts, ends=p.ends, rows=p.rows, positions=p.positions, slots=p.slots)
    for k, v in got.items():
        assert np.array_equal(v.numpy(), want[k]), k
    assert int(p.free_count) == int(count) == want["left"]


def test_plan_without_room_names_the_rows():
    tables = torch.full((3, 4), -1, dtype=I32)
    with pytest.raises(RuntimeError, match=r"rows \[1, 2\]"):
        kvcache.plan_tokens(tables, ints([0, 0, 0]), ints([16, 33, 1]), ints([4, 5, 6]), ints([3]), 16, 50)


def _append_case(seed, dim, heads, block):
    g = torch.Generator().manual_seed(seed)
    codes = C.random_codes((2, 9, heads, block, dim), seed)
    scale = torch.exp2(torch.randint(-12, -5, (2, 9, heads), generator=g).float())
    # block 3 from its start over its end into block 5, one token deep in block 1, a skipped token, one growing block 7
    slots = [3 * block + i for i in range(block)] + [5 * block + i for i in range(min(7, block))] + [1 * block + 5, -1, 7 * block + block - 1]
    n = len(slots)
    x = torch.randn(2, n, heads, dim, generator=g) * torch.exp2(torch.randint(-6, 3, (2, n, heads, 1), generator=g).float())
    x[:, -1] *= 40
    x = x.bfloat16()
    x[0, 1, 0, 3], x[1, 2, 0, 1], x[1, 2, 0, 2] = math.inf, math.nan, -math.inf
    x[:, block + 1] = 0
    return codes, scale, x, slots


@pytest.mark.parametrize("dim,heads,block", [(64, 1, 16), (128, 3, 32), (64, 2, 128)])
def test_append(dim, heads, block):
    codes, scale, x, slots = _append_case(5, dim, heads, block)
    want, wscale = O.append(C.values(codes), scale.numpy(), x[0].float().numpy(), x[1].float().numpy(), slots)
    kvcache.append(codes, scale, x[0], x[1], ints(slots))
    assert np.array_equal(C.values(codes), want, equal_nan=True) and np.array_equal(scale.double().numpy(), wscale)


def test_scale_for_borders():
    a = torch.tensor([0.0, 448.0, 449.0, 224.0, 1.0, 3.3e38, 1e-38, 448 * 2.0 ** -118, 1.75, 1.7578125])
    got = kvcache.scale_for(a).double().tolist()
    assert got == [O.scale_for(float(v)) for v in a.double()]


@pytest.mark.parametrize("case", C.ATTENTION[:9])
def test_attention(case):
    d = C.attention_inputs(case)
    q = d["q"][: d["T"], 1: 1 + d["hq"]]
    got = kvcache.paged_attention(q, d["codes"], d["scale"], d["tables"], d["starts"], d["ends"]).double().numpy()
    want, A = O.attention(q.float().numpy(), C.values(d["codes"]), d["scale"].double().numpy(), d["tables"].numpy(), d["starts"].numpy(), d["ends"].numpy(), d["dim"] ** -0.5)
    # fp32: a score of magnitude S is off by a few times 2^-24 S sqrt(D), S <= 40 here; the weights by as much, relatively
    assert np.all(np.abs(got - want) <= 2.0 ** -24 * (4 * 40 * d["dim"] ** 0.5 + d["codes"].shape[1] * d["block"] ** 0.5) * A + 1e-30)


def test_attention_token_that_sees_nothing_is_zero():
    kv, scale = C.random_codes((2, 2, 1, 16, 64), 1), torch.ones(2, 2, 1)
    o = kvcache.paged_attention(torch.randn(2, 1, 64), kv, scale, ints([[0]]), ints([0, 2]), ints([0]))
    assert torch.equal(o, torch.zeros(2, 1, 64))


@pytest.mark.parametrize("requests,beams,vocab", [(1, 1, 5), (3, 4, 7), (2, 8, 100), (2, 3, 2)])
@pytest.mark.parametrize("finish", [False, True])
def test_select(requests, beams, vocab, finish):
    g = torch.Generator().manual_seed(beams)
    x = torch.randn(requests, beams, vocab, generator=g).bfloat16()
    x[0, 0, 1] = math.nan
    scores = -torch.rand(requests, beams, generator=g)
    scores[:, beams // 2 + 1:] = -math.inf
    fin = torch.rand(requests, beams, generator=g) < 0.4 if finish else None
    s, p, t, done = beam.beam_select(x, scores, fin, 1 if finish else None)
    for r, row in enumerate(O.select(x, scores, fin, 1 if finish else None)):
        assert [(int(a), int(b)) for a, b in zip(p[r], t[r])] == [(b, v) for _, b, v in row]
        assert np.allclose(s[r].numpy(), [v for v, _, _ in row], rtol=2.0 ** -23)
        for k in range(beams):
            assert bool(done[r, k]) == (finish and (bool(fin[r, p[r, k]]) or int(t[r, k]) == 1))


def test_reorder():
    lens = [40, 40, 40, 32, 32, 32]
    tables, blocks, left = C.paged(lens, 16, 2, spare_blocks=6)
    codes = C.random_codes((2, 2, blocks, 2, 16, 64), 4)
    scale = torch.rand(2, 2, blocks, 2)
    parents = np.array([[1, 1, 2], [2, 0, 0]], dtype=np.int32)
    want = O.reorder(C.values(codes), scale.numpy(), tables, lens, parents, left)
    t, n, s = beam.beam_reorder(codes, scale, torch.from_numpy(tables), ints(lens), torch.from_numpy(parents), ints(left.tolist()))
    for a, b in zip((C.values(codes), scale.numpy(), t.numpy(), n.numpy(), s.numpy()), want):
        assert np.array_equal(a, b)


# ------------------------------------------------------------------------------------------------ refusals
def _layer(blocks=4, heads=2, block=16, dim=64):
    return torch.zeros(2, blocks, heads, block, dim, dtype=torch.uint8).view(C.F8), torch.zeros(2, blocks, heads)


def test_refusals_of_the_cache():
    for kw in (dict(block=8), dict(head_dim=96), dict(rows=0), dict(rows=kvcache.MAX_ROWS + 1), dict(blocks=1 << 28), dict(layers=0), dict(max_len=0)):
        with pytest.raises(ValueError):
            kvcache.PagedKVCache(**{**dict(layers=1, kv_heads=1, head_dim=64, blocks=4, rows=2, max_len=32, device="meta" if kw.get("blocks") else "cpu"), **kw})
    with pytest.raises(ValueError, match="spare"):
        kvcache.PagedKVCache(1, 1, 64, 4, 2, 32, device="cpu").reorder(ints([[0, 0]]))


def test_refusals_of_plan():
    ok = dict(tables=torch.full((2, 3), -1, dtype=I32), lengths=ints([0, 0]), new_lens=ints([1, 1]), free=ints([0, 1]), free_count=ints([2]), block=16, tokens=2)
    bad = [dict(tables=ok["tables"].long()), dict(tables=ok["tables"][:, :2]), dict(lengths=ints([0])), dict(new_lens=ok["new_lens"].float()), dict(free_count=ints([1, 1])),
           dict(block=0), dict(tokens=-1), dict(free=ints([0, 1]).to(torch.int64)), dict(free_count_out=torch.zeros(1)), dict(block=1 << 30)]
    for b in bad:
        with pytest.raises(ValueError):
            kvcache.plan_tokens(**{**ok, **b})


def test_refusals_of_append():
    kv, scale = _layer()
    k = torch.zeros(3, 2, 64)
    ok = dict(kv=kv, scale=scale, k=k, v=k, slots=ints([0, 1, 2]))
    odd, oscale = _layer(block=24)
    bad = [dict(kv=kv.view(torch.uint8)), dict(kv=kv[:, :2]), dict(kv=odd, scale=oscale), dict(scale=scale.double()), dict(scale=scale[:, :2]), dict(k=k[:, :1]), dict(v=k[:2]), dict(k=torch.zeros(3, 2, 32)),
           dict(slots=ints([0, 1])), dict(slots=torch.zeros(3))]
    for b in bad:
        with pytest.raises(ValueError):
            kvcache.append(**{**ok, **b})


def test_refusals_of_attention():
    kv, scale = _layer()
    ok = dict(q=torch.zeros(2, 4, 64), kv=kv, scale=scale, tables=ints([[0, 1]]), starts=ints([0, 2]), ends=ints([5]))
    bad = [dict(q=torch.zeros(2, 3, 64)), dict(q=torch.zeros(2, 4, 32)), dict(starts=ints([0])), dict(ends=ints([1, 1])), dict(tables=ints([0, 1])), dict(ends=torch.ones(1)), dict(max_new=0),
           dict(tables=ints([[7, 1]])), dict(tables=ints([[-1, 1]]))]
    for b in bad:
        with pytest.raises(ValueError):
            kvcache.paged_attention(**{**ok, **b})


def test_refusals_of_beams():
    x, s = torch.zeros(2, 3, 5), torch.zeros(2, 3)
    bad = [dict(logits=x[0]), dict(scores=s.double()), dict(scores=s[:, :2]), dict(eos=5), dict(finished=torch.zeros(2, 3, dtype=torch.bool)), dict(finished=torch.zeros(2, 3), eos=1),
           dict(logits=torch.zeros(1, 33, 40), scores=torch.zeros(1, 33))]
    for b in bad:
        with pytest.raises(ValueError):
            beam.beam_select(**{**dict(logits=x, scores=s), **b})
    kv, scale = (t[None] for t in _layer(6))
    ok = dict(kv=kv, scale=scale, tables=ints([[0, -1], [1, -1]]), lengths=ints([3, 3]), parents=ints([[1, 1]]), spare=ints([2, 3]))
    bad = [dict(kv=kv[0]), dict(scale=scale[0]), dict(parents=ints([[1, 1, 1]])), dict(parents=ints([[2, 0]])), dict(spare=ints([2])), dict(spare=ints([-1, 3])), dict(lengths=ints([3])),
           dict(tables_out=ok["tables"]), dict(spare_out=ok["spare"])]
    for b in bad:
        with pytest.raises(ValueError):
            beam.beam_reorder(**{**ok, **b})
