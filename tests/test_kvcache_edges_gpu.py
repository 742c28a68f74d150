"""Paged 8-bit cache and beam search on the GPU at the borders of what their calls allow."""
import numpy as np
import pytest
import torch

import kv_oracle as O

pytestmark = pytest.mark.gpu
I32 = torch.int32


def ints(v):
    return torch.tensor(v, dtype=I32, device="cuda")


def clean():
    from noeira_b200.ops import check_status
    torch.cuda.synchronize()
    check_status()


def reported(match):
    from noeira_b200.ops import check_status
    from noeira_b200.ops.status import DeviceStatusError
    with pytest.raises(DeviceStatusError, match=match):
        check_status()


# ------------------------------------------------------------------------------------------------ plan
@pytest.mark.parametrize("lengths,new,width,free,tokens", [
    ([0, 0, 0, 5], [16, 33, 1, 3], 4, 3, 60),          # too few blocks
    ([0, 60, 0], [10, 10, 10], 4, 9, 30),              # a row outgrows its table
    ([64, 3], [1, 1], 4, 9, 2),                        # a full row
    ([0, 0, 0], [10, 10, 10], 4, 9, 25),               # the token dimension is too short
    ([-5, 3, 0], [2, -2, 4], 4, 9, 30),                # lengths that are none
    ([0, 0, 7], [0x7fffffff, 0x7fffffff, 1], 4, 9, 8),  # sums past 32 bits
])
def test_tokens_of_refused_rows_have_place_zero(lengths, new, width, free, tokens):
    """What is looked up by position (a table of learned positions) is looked up before anyone reads the status word."""
    from noeira_b200.ops import kvcache
    tables = np.full((len(lengths), width), -1, dtype=np.int32)
    for i, n in enumerate(lengths):
        tables[i, : max(0, -(-n // 16))] = 50 + 4 * i + np.arange(max(0, -(-n // 16)))
    stack = np.arange(free) + 10
    want, refused = O.plan(tables, lengths, new, stack, free, 16, tokens)
    assert refused
    p = kvcache.plan_tokens(torch.from_numpy(tables).cuda(), ints(lengths), ints(new), ints(stack.tolist()), ints([free]), 16, tokens)
    reported("no room")
    slots, positions = p.slots.cpu().numpy(), p.positions.cpu().numpy()
    assert np.array_equal(slots, want["slots"]) and np.array_equal(p.rows.cpu().numpy(), want["rows"])
    assert np.array_equal(positions, np.where(want["slots"] >= 0, want["positions"], 0))
    assert positions.min() >= 0 and positions.max() < width * 16


@pytest.mark.parametrize("block", [16, 32])
def test_rows_hold_max_len_tokens_and_no_more(block):
    """A length that is no multiple of the block: the last block has places behind it, which belong to no token."""
    from noeira_b200.ops import kvcache
    c = kvcache.PagedKVCache(1, 1, 64, 8, 2, 18, block)
    p = c.plan(ints([18, 17]), 35)
    clean()
    assert p.positions.tolist() == list(range(18)) + list(range(17)) and min(p.slots.tolist()) >= 0
    p = c.plan(ints([1, 1]), 2)
    reported("no room")
    assert p.positions.tolist() == [0, 17] and p.slots.tolist()[0] == -1 and c.lengths.tolist() == [18, 18]
    p = c.plan(ints([0, 10]), 10)
    reported("no room")
    assert p.positions.tolist() == [0] * 10 and p.slots.tolist() == [-1] * 10 and c.lengths.tolist() == [18, 18]


@pytest.mark.parametrize("bad", [8, 1 << 27, 1 << 28, 0x7fffffff, -1, -(1 << 31)])
@pytest.mark.parametrize("place", ["table", "stack"])
def test_plan_reports_blocks_that_are_none(bad, place):
    """An id shifted past 32 bits would be the slot of another block."""
    from noeira_b200.ops import kvcache
    c = kvcache.PagedKVCache(1, 1, 64, 8, 2, 64, 16)
    c.plan(ints([5, 5]), 10)                                # blocks 0 and 1
    clean()
    if place == "table":
        c.tables[0, 0] = bad
        want = [-1] * 11 + [32, 33] + [21, 22, 23]          # row 0's tokens 5 to 15 lie in its first block, then block 2
    else:
        c.free[int(c.free_count) - 1] = bad
        want = list(range(5, 16)) + [-1, -1] + [21, 22, 23]
    p = c.plan(ints([13, 3]), 16)
    reported("bounds")
    assert p.slots.tolist() == want
    assert p.positions.tolist() == [q if s >= 0 else 0 for q, s in zip([*range(5, 18), *range(5, 8)], want)]
    assert c.tables[0, 1].item() == (2 if place == "table" else -1)
    k = torch.ones(16, 1, 64, dtype=torch.bfloat16, device="cuda")
    before = c.kv.clone()
    c.append(0, k, k, p)
    clean()
    changed = (c.kv.view(torch.uint8) != before.view(torch.uint8)).any(-1)[0].any(0)[:, 0].reshape(-1).nonzero().reshape(-1).tolist()
    assert changed == sorted(s for s in want if s >= 0)


# ------------------------------------------------------------------------------------------------ append
def gaps(kind, block):
    """Slots of a call that leaves places of a block out."""
    b = [7 * block, 2 * block, 11 * block, 4 * block, 9 * block]
    if kind == "every second":
        return [s + i for s in b for i in range(0, block, 2)]
    if kind == "from the middle":
        return [b[0] + 3, b[0] + 5, b[1] + 1, b[2] + 2, b[2] + 3, b[2] + block - 1, b[3] + block - 1, b[4], b[4] + block - 1]
    if kind == "behind skipped tokens":
        return [b[0], -1, b[0] + 2, -1, 1 << 30, b[0] + 3, -1, b[0] + 9, b[1] + 4, -1, b[1] + 6] + [-1] * 40 + [b[1] + 8, b[2] + 1, b[3] + 1]
    return [s + i for s in b for i in range(block) if i % 5] + list(range(20 * block, 20 * block + 1100))     # more than a short call's


@pytest.mark.parametrize("kind", ["every second", "from the middle", "behind skipped tokens", "many"])
@pytest.mark.parametrize("block", [16, 128])
@pytest.mark.parametrize("dim,heads", [(64, 3), (128, 1)])
@pytest.mark.parametrize("growing", [False, True])
def test_append_leaves_places_out(kind, block, dim, heads, growing):
    """The scale of a block is one for all tokens of the call, wherever the places between them are."""
    import kv_cases as C
    from noeira_b200.ops import kvcache
    slots = gaps(kind, block)
    n, blocks = len(slots), 20 + -(-1100 // block)
    g = torch.Generator().manual_seed(block + dim)
    codes, scale = C.random_codes((2, blocks, heads, block, dim), 5), torch.exp2(torch.randint(-12, -5, (2, blocks, heads), generator=g).float())
    x = torch.randn(2, n, heads, dim, generator=g)
    if growing:
        x *= 1.5 ** (torch.arange(n) % 24)[None, :, None, None]
    x = x.bfloat16()
    want, wscale = O.append(C.values(codes), scale.numpy(), x[0].float().numpy(), x[1].float().numpy(), slots)
    c, sc = codes.cuda(), scale.cuda()
    kvcache.append(c, sc, x[0].cuda(), x[1].cuda(), ints(slots))
    clean()
    assert np.array_equal(sc.cpu().double().numpy(), wscale) and np.array_equal(C.values(c), want, equal_nan=True)
    kvcache.append(codes, scale, x[0], x[1], torch.tensor(slots, dtype=I32))
    assert torch.equal(codes.view(torch.uint8), c.cpu().view(torch.uint8))


@pytest.mark.parametrize("whole", [True, False])
def test_captured_steps_with_reorders(whole):
    """A step captured with its reorder, and one captured without it and replayed between eager reorders, leave the cache as eager
    steps do."""
    from noeira_b200.ops import kvcache
    g = torch.Generator().manual_seed(7)
    beams, heads, rows = 3, 2, 6
    caches = [kvcache.PagedKVCache(1, heads, 64, blocks=50, rows=rows, max_len=60, block=16, spares=True) for _ in range(2)]
    first = ints([21, 0, 0, 16, 0, 0])
    kv = torch.randn(37, 2 * heads, 64, generator=g).bfloat16().cuda()
    for c in caches:
        c.append(0, kv[:, :heads], kv[:, heads:], c.plan(first, 37))
        c.reorder(torch.zeros(2, beams, dtype=I32, device="cuda"))
        c.refill_spares()
    x, parents, one = torch.zeros(rows, 2 * heads, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, beams, dtype=I32, device="cuda"), ints([1] * rows)
    q = torch.randn(rows, heads, 64, generator=g).bfloat16().cuda()

    def step(c, reorder=True):
        p = c.plan(one, rows)
        c.append(0, x[:, :heads], x[:, heads:], p)
        o = c.attend(0, q, p, max_new=1)
        if reorder:
            c.reorder(parents)
        return o

    eager, captured = caches
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        out = step(captured, whole)
    for _ in range(25):
        x.copy_(torch.randn(rows, 2 * heads, 64, generator=g))
        parents.copy_(torch.randint(0, beams, (2, beams), generator=g))
        want = step(eager)
        graph.replay()
        if not whole:
            captured.reorder(parents)
        clean()
        assert torch.equal(out, want)
        for a, b in ((eager.tables, captured.tables), (eager.lengths, captured.lengths), (eager.spare, captured.spare), (eager.free_count, captured.free_count),
                     (eager.scale, captured.scale), (eager.kv.view(torch.uint8), captured.kv.view(torch.uint8))):
            assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ beams
def logits_of(kind, beams, vocab):
    """Different logits of one value in 64 bits; beam 0 is the one that counts."""
    v = torch.arange(vocab).float()
    x = torch.stack([torch.sin(v * (b + 1)) for b in range(beams)])
    if kind == "infinite":
        x[0, vocab // 2] = float("inf")
    if kind == "infinite twice":
        x[0, vocab - 1] = x[0, vocab // 3] = float("inf")
    if kind == "near zero":                                   # rising, far below what a value of size log(vocab) can tell
        x = (v * 2.0 ** -90).expand(beams, vocab).clone()
        x[:, vocab - 1] = 1.0
    if kind == "few":                                         # fewer finite logits than beams, and two of them equal
        x[0] = float("-inf")
        x[0, vocab - 1], x[0, vocab // 2], x[0, vocab // 3] = 2.0, 2.0, float("nan")
    return x


@pytest.mark.parametrize("kind", ["infinite", "infinite twice", "near zero", "few", "plain"])
@pytest.mark.parametrize("beams,vocab", [(2, 4), (4, 4), (4, 5), (8, 20011), (32, 300), (5, 49152)])
@pytest.mark.parametrize("fp32", [False, True])
def test_select_equal_values_of_different_logits(kind, beams, vocab, fp32):
    from noeira_b200.ops import beam
    inf = float("inf")
    x = logits_of(kind, beams, vocab)
    x = x if fp32 else x.bfloat16()
    # one beam alone; a far score, at which all its logits are one; none; a beam that is finished at -inf, one that is at 0
    scores = torch.full((6, beams), -inf)
    scores[0, 0], scores[1, 0], scores[2, 0], scores[4, beams - 1] = 0.0, -1e25, float("nan"), 0.0
    scores[5] = 0.0
    x = x.expand(6, beams, vocab).contiguous()
    fin = torch.zeros(6, beams, dtype=torch.bool)
    fin[3, 0] = fin[4, beams - 1] = True
    for finished, eos in ((None, None), (fin, vocab - 1), (fin, vocab // 2)):
        s, p, t, _ = beam.beam_select(x.cuda(), scores.cuda(), None if finished is None else finished.cuda(), eos)
        clean()
        for r, row in enumerate(O.select(x, scores, finished, eos)):
            assert [(int(a), int(b)) for a, b in zip(p[r], t[r])] == [(b, v) for _, b, v in row], r
        c = beam.beam_select(x, scores, finished, eos)
        assert torch.equal(p.cpu(), c[1]) and torch.equal(t.cpu(), c[2])


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("pad", [0, 1])
def test_select_takes_every_number_of_beams(fp32, pad):
    """In ascending order: none may depend on what a larger one has set up before it.  Rows enough for long parts."""
    from noeira_b200.ops import beam
    vocab = 9000
    g = torch.Generator(device="cuda").manual_seed(2)
    for beams in range(1, 33):
        rows = -(-160 // beams)
        wide = torch.randn(rows, beams, vocab + pad, generator=g, device="cuda")
        x = (wide if fp32 else wide.bfloat16())[..., :vocab]
        s, p, t, _ = beam.beam_select(x, torch.zeros(rows, beams, device="cuda"))
        clean()
        value = torch.log_softmax(x.double(), -1)
        assert torch.equal(torch.sort(s, 1, descending=True).values, s) and bool((p < beams).all())
        # fp32 sums of exponentials of 2^-22 each, their logarithm, and the value's own rounding
        assert bool(((value.gather(2, t.long().clamp(0, vocab - 1)[:, None].expand(rows, beams, beams)).gather(1, p.long()[:, None])[:, 0] - s).abs() <= 2.0 ** -20 + 2.0 ** -24 * 40).all())
        top = value.reshape(rows, -1).topk(beams).values
        assert bool(((top - s).abs() <= 2.0 ** -20 + 2.0 ** -24 * 40).all())


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("tokens", [200, 1])
def test_attention_over_a_million_keys(tokens):
    """One row's tiles walk more than 2^24 steps between them.  Its table names four blocks again and again, so the definition is a
    sum over 512 keys, each as often as the token sees it."""
    from noeira_b200.ops import kvcache
    import kv_cases as C
    hq, hk, dim, block, keys = 32, 8, 128, 128, 1 << 20
    g = torch.Generator(device="cuda").manual_seed(3)
    codes = C.random_codes((2, 4, hk, block, dim), 3).cuda()
    scale = torch.exp2(torch.randint(-10, -6, (2, 4, hk), generator=torch.Generator().manual_seed(4)).float()).cuda()
    table = (torch.arange(keys // block, device="cuda") % 4).to(I32)[None].contiguous()
    q = torch.randn(tokens, hq, dim, device="cuda", generator=g).bfloat16()
    out = kvcache.paged_attention(q, codes, scale, table, ints([0, tokens]), ints([keys]))
    clean()
    k, v = ((codes[w].double() * scale[w].double()[..., None, None]).transpose(0, 1).reshape(hk, -1, dim).repeat_interleave(hq // hk, 0) for w in (0, 1))
    s = q.double().transpose(0, 1) @ k.transpose(1, 2) * dim ** -0.5
    sees = keys - tokens + 1 + torch.arange(tokens, device="cuda")
    times = (sees[:, None] - torch.arange(4 * block, device="cuda") + 4 * block - 1) // (4 * block)
    p = torch.exp(s - s.amax(-1, keepdim=True)) * times
    p = p / p.sum(-1, keepdim=True)
    want, A = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
    # as for shorter rows; the sums of a warp's piece: two weights and a product of 16 keys per step, one after the other
    piece = -(-((tokens * 4 + 15) // 16) * hk * (keys // 16 + 2) // (148 * 4 * 3))
    S = dim ** -0.5 * float((q.double().abs().sum(-1)).max() * k.abs().max())
    most = 2.0 ** -8 * want.abs() + A * (2.0 ** -8 + 2 * (2.0 ** -24 * dim * S + 2.0 ** -21) + 2.0 ** -24 * 3 * (piece + 1776))
    err = (out.double() - want).abs()
    assert bool((err <= most).all()), float((err / most).max())


@pytest.mark.parametrize("tokens,dim", [(130, 128), (100, 128), (130, 64), (1, 128)])
def test_attention_through_very_wide_tables(tokens, dim):
    """Tables with room for so many keys that steps are counted in 64 bits: the bits are those of narrow tables."""
    from noeira_b200.ops import kvcache
    import kv_cases as C
    hq, hk, block = 32, 8, 128
    held, new = [3000, 900, 4000, 17], [tokens, 1, 1, 2]
    d = C.attention_inputs((held, new, hq, hk, dim, block))
    q = d["q"][: d["T"], 1: 1 + hq].contiguous().cuda()
    width = (1 << 30) // block
    wide = torch.full((4, width), -1, dtype=I32, device="cuda")
    wide[:, : d["tables"].shape[1]] = d["tables"].cuda()
    rest = (d["starts"].cuda(), d["ends"].cuda(), d["max_new"])
    a = kvcache.paged_attention(q, d["codes"].cuda(), d["scale"].cuda(), d["tables"].cuda(), *rest)
    b = kvcache.paged_attention(q, d["codes"].cuda(), d["scale"].cuda(), wide, *rest)
    clean()
    assert torch.equal(a, b)


def test_attention_counts_more_than_32_bits_of_steps():
    """4200 rows of one token over the same million keys: 2.2e9 steps.  Every token sees every key, so the definition is the
    softmax over the 512 different ones."""
    from noeira_b200.ops import kvcache
    import kv_cases as C
    rows, hq, hk, dim, block, keys = 4200, 32, 8, 128, 128, 1 << 20
    codes = C.random_codes((2, 4, hk, block, dim), 3).cuda()
    scale = torch.exp2(torch.randint(-10, -6, (2, 4, hk), generator=torch.Generator().manual_seed(4)).float()).cuda()
    table = (torch.arange(keys // block, device="cuda") % 4).to(I32)[None].repeat(rows, 1)
    q = torch.randn(rows, hq, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).bfloat16()
    out = kvcache.paged_attention(q, codes, scale, table, torch.arange(rows + 1, dtype=I32, device="cuda"), ints([keys] * rows), max_new=1)
    clean()
    k, v = ((codes[w].double() * scale[w].double()[..., None, None]).transpose(0, 1).reshape(hk, -1, dim).repeat_interleave(hq // hk, 0) for w in (0, 1))
    p = torch.softmax(q.double().transpose(0, 1) @ k.transpose(1, 2) * dim ** -0.5, -1)
    want, A = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
    # a warp's sums over one job, which is shorter than its piece
    S = dim ** -0.5 * float((q.double().abs().sum(-1)).max() * k.abs().max())
    most = 2.0 ** -8 * want.abs() + A * (2.0 ** -8 + 2 * (2.0 ** -24 * dim * S + 2.0 ** -21) + 2.0 ** -24 * 3 * (keys // 16))
    err = (out.double() - want).abs()
    assert bool((err <= most).all()), float((err / most).max())


def test_attention_reports_starts_that_are_none():
    """Rows that all claim all tokens have more steps than their sizes allow: refused as a whole."""
    from noeira_b200.ops import kvcache
    rows, tokens, block = 4096, 60, 128
    kv, scale = torch.zeros(2, 1, 1, block, 128, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn), torch.ones(2, 1, 1, device="cuda")
    q = torch.ones(tokens, 16, 128, dtype=torch.bfloat16, device="cuda")
    starts = ints([0, tokens] * (rows // 2) + [0])
    out = torch.full_like(q, 7)
    kvcache.paged_attention(q, kv, scale, torch.zeros(rows, 8192, dtype=I32, device="cuda"), starts, ints([1 << 20] * rows), out=out)
    reported("bounds")
    assert bool((out == 7).all())


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("held,new,dim,power", [([700, 5], [1, 1], 64, 30), ([90], [1], 128, 24), ([3000, 40], [3, 17], 128, 40), ([60, 2100, 0], [500, 1, 300], 128, 27),
                                                ([16, 700], [600, 257], 64, 40), ([5000, 31, 2], [1, 1, 1], 64, 21)])
def test_attention_of_far_scores(mode, held, new, dim, power):
    """Scores of 2^20 to 2^45: what rounding leaves of a maximum must not become a weight.  Where the largest score leads by more
    than any rounding of it, the output is that key's value."""
    import kv_cases as C
    from noeira_b200.ops import kvcache
    hq, hk, block = 8, 2, 32
    d = C.attention_inputs((held, new, hq, hk, dim, block), seed=power)
    g = torch.Generator().manual_seed(power)
    scale = torch.exp2(torch.randint(-9, -5, d["scale"].shape, generator=g).float())
    scale[0] *= torch.exp2(torch.randint(power - 3, power + 1, scale.shape[1:], generator=g).float())
    q, codes = d["q"][: d["T"], 1: 1 + hq].contiguous().cuda(), d["codes"].cuda()
    old = kvcache.set_attention_mode(mode)
    try:
        out = kvcache.paged_attention(q, codes, scale.cuda(), d["tables"].cuda(), d["starts"].cuda(), d["ends"].cuda(), max_new=d["max_new"])
        clean()
    finally:
        kvcache.set_attention_mode(old)
    assert bool(torch.isfinite(out).all())
    scale, st, clear = scale.cuda().double(), d["starts"].tolist(), 0
    for i, end in enumerate(d["ends"].tolist()):
        a, b = st[i], st[i + 1]
        ids = d["tables"][i, : -(-end // block)].long().cuda()
        k, v = ((codes[w, ids].double() * scale[w, ids][..., None, None]).transpose(0, 1).reshape(hk, -1, dim)[:, :end].repeat_interleave(hq // hk, 0) for w in (0, 1))
        see = torch.arange(end, device="cuda")[None] <= (end - (b - torch.arange(a, b, device="cuda")))[:, None]
        s = (q[a:b].double().transpose(0, 1) @ k.transpose(1, 2) * dim ** -0.5).masked_fill(~see, float("-inf"))
        first, at = s.topk(min(2, end), -1)
        off = 2.0 ** -24 * (dim + 4) * dim ** -0.5 * q[a:b].double().abs().transpose(0, 1) @ k.abs().amax(1)[..., None]      # of one score
        lead = (first[..., 0] - first[..., -1] if end > 1 else torch.full_like(first[..., 0], 1e30))
        lead = torch.where(torch.isnan(lead), torch.full_like(lead, 1e30), lead)                                            # a token that sees one key
        leads = lead > 2 * off[..., 0] + 40                                                                                 # e^-40 of 2^45 keys is nothing
        want = v.gather(1, at[..., :1].expand(-1, -1, dim)).transpose(0, 1)
        got, leads = out[a:b].double(), leads.transpose(0, 1)
        clear += int(leads.sum())
        assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 1e-9 * v.abs().max())[leads].all())
    assert clear > 0.5 * d["T"] * hq


@pytest.mark.parametrize("held,new,hq,hk,dim", [([3000, 17], [1, 1], 8, 2, 64), ([300, 0, 40], [20, 1, 33], 32, 8, 128), ([500, 0, 0], [700, 300, 1], 16, 8, 64)])
@pytest.mark.parametrize("power", [0, 30])
def test_attention_in_place(held, new, hq, hk, dim, power):
    """``out`` may be ``q``, also where far scores make the rows of prompts be done over."""
    import kv_cases as C
    from noeira_b200.ops import kvcache
    d = C.attention_inputs((held, new, hq, hk, dim, 32))
    d["scale"][0] *= 2.0 ** power
    wide = torch.zeros(d["T"], 3 * hq, dim, dtype=torch.bfloat16, device="cuda")          # a packed projection's queries
    wide[:, :hq] = d["q"][: d["T"], 1: 1 + hq].cuda()
    q = wide[:, :hq]
    rest = (d["codes"].cuda(), d["scale"].cuda(), d["tables"].cuda(), d["starts"].cuda(), d["ends"].cuda(), d["max_new"])
    want = kvcache.paged_attention(q, *rest)
    got = kvcache.paged_attention(q, *rest, out=q)
    clean()
    assert got.data_ptr() == wide.data_ptr() and torch.equal(got, want) and bool((wide[:, hq:] == 0).all())
