"""Paged 8-bit cache, attention over it and beam search on the GPU, against definitions in 64 bits.

Tolerances of attention.  The output is rounded to bf16 (2^-8 of its value).  A weight of the softmax is rounded once before it
multiplies the values: to bf16 at most (2^-8), which moves the output by at most 2^-8 A, A the same weighted mean of |v|.  A score
s = c q k is a sum in fp32 of exact products: off by at most 2^-24 D sum|c q k|, and the exponential by 2^-21 more; S bounds
sum|c q k| over the rows.  The sums over n keys add 2^-24 n at most.
"""
import math

import numpy as np
import pytest
import torch

import kv_cases as C
import kv_oracle as O

pytestmark = pytest.mark.gpu
I32 = torch.int32


def ints(v):
    return torch.tensor(v, dtype=I32, device="cuda")


def clean():
    from noeira_b200.ops import check_status
    torch.cuda.synchronize()
    check_status()


# ------------------------------------------------------------------------------------------------ plan
@pytest.mark.parametrize("lengths,new,block,spare,pad", C.PLANS)
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(lengths, new, block, spare, pad, in_place):
    from noeira_b200.ops import kvcache
    tables, blocks, left = C.paged(lengths, block, 3, spare_blocks=sum(-(-n // block) + 1 for n in new) + spare, extra_width=-(-max(new) // block) + 1)
    tokens = sum(new) + pad
    want, refused = O.plan(tables, lengths, new, left, len(left), block, tokens)
    assert not refused
    t, count = torch.from_numpy(tables).cuda(), ints([len(left)])
    out = None if in_place else ints([-5])
    p = kvcache.plan_tokens(t, ints(lengths), ints(new), ints(left.tolist()), count, block, tokens, free_count_out=out)
    clean()
    for k, v in dict(tables=t, starts=p.starts, ends=p.ends, rows=p.rows, positions=p.positions, slots=p.slots).items():
        assert np.array_equal(v.cpu().numpy(), want[k]), k
    assert int(p.free_count) == want["left"] and int(count) == (want["left"] if in_place else len(left))


@pytest.mark.parametrize("lengths,new,width,free,tokens", [
    ([0, 0, 0, 5], [16, 33, 1, 3], 4, 3, 60),          # the second finds too few blocks, the third needs one, the fourth none
    ([0, 60, 0], [10, 10, 10], 4, 9, 30),              # the second outgrows its table
    ([0, 0, 0], [10, 10, 10], 4, 9, 25),               # the third outgrows the token dimension
    ([-1, 3, 0], [1, -2, 4], 4, 9, 30),                # lengths that are none
    ([0, 0, 7], [0x7fffffff, 0x7fffffff, 1], 4, 9, 8),  # sums past 32 bits
])
def test_plan_refuses_rows(lengths, new, width, free, tokens):
    from noeira_b200.ops import check_status, kvcache
    from noeira_b200.ops.status import DeviceStatusError
    rows = len(lengths)
    tables = np.full((rows, width), -1, dtype=np.int32)
    for i, n in enumerate(lengths):
        tables[i, : max(0, -(-n // 16))] = 50 + 4 * i + np.arange(max(0, -(-n // 16)))
    stack = np.arange(free) + 10
    want, refused = O.plan(tables, lengths, new, stack, free, 16, tokens)
    assert refused
    t = torch.from_numpy(tables).cuda()
    p = kvcache.plan_tokens(t, ints(lengths), ints(new), ints(stack.tolist()), ints([free]), 16, tokens)
    with pytest.raises(DeviceStatusError, match="no room"):
        check_status()
    for k, v in dict(tables=t, ends=p.ends, slots=p.slots).items():
        assert np.array_equal(v.cpu().numpy(), want[k]), k
    assert np.array_equal(p.starts.cpu().numpy(), np.minimum(want["starts"], 0x7fffffff)) and int(p.free_count) == want["left"]


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("dim,heads", [(64, 1), (64, 5), (128, 3)])
@pytest.mark.parametrize("layout", ["packed", "odd"])
def test_append(dim, heads, block, layout):
    from noeira_b200.ops import kvcache
    g = torch.Generator().manual_seed(block + dim)
    codes = C.random_codes((2, 40, heads, block, dim), 5)
    scale = torch.exp2(torch.randint(-12, -5, (2, 40, heads), generator=g).float())
    # runs of many kinds: whole blocks, starts and ends inside a block, one token, tokens that are skipped
    ids = torch.randperm(40, generator=g).tolist()
    slots = []
    for off, n in ((0, 2 * block + 3), (block - 1, 1), (5, 1), (0, 1), (block // 2, block), (3, 2), (0, 5), (block - 2, block + 9)):
        page, at = [ids.pop() for _ in range(4)], off
        slots += [page[(at + i) // block] * block + (at + i) % block for i in range(n)]
    slots = slots[:9] + [-1] + slots[9:40] + [40 * block, 0x7fffffff, -7] + slots[40:]
    n = len(slots)
    x = torch.randn(2, n, heads, dim, generator=g) * torch.exp2(torch.randint(-8, 3, (2, n, 1, 1), generator=g).float())
    x[0, 1, 0, 3], x[1, 2, 0, 1], x[1, 3, 0, 2] = math.inf, math.nan, -math.inf
    x[:, 5:7] = 0
    x = x.bfloat16()
    want, wscale = O.append(C.values(codes), scale.numpy(), x[0].float().numpy(), x[1].float().numpy(), slots)
    if layout == "packed":
        buf = torch.zeros(n, 2 * heads + 3, dim, dtype=torch.bfloat16, device="cuda")
        k, v = buf[:, 3: 3 + heads], buf[:, 3 + heads:]
    else:                                              # rows that begin on no 16-byte boundary
        buf = torch.zeros(2, n, heads * dim + 3, dtype=torch.bfloat16, device="cuda")
        k, v = (b[:, 1: 1 + heads * dim].unflatten(1, (heads, dim)) for b in buf)
    k.copy_(x[0])
    v.copy_(x[1])
    codes, scale, slots = codes.cuda(), scale.cuda(), ints(slots)
    for _ in range(2):                                 # the second call finds what the first one wrote and changes nothing
        kvcache.append(codes, scale, k, v, slots)
        clean()
        assert np.array_equal(scale.cpu().double().numpy(), wscale)
        assert np.array_equal(C.values(codes), want, equal_nan=True)


def test_append_many_tokens_in_steps_equals_the_cpu_form():
    """A prompt and single tokens after it, the values growing, so that scales have to be raised again and again."""
    from noeira_b200.ops import kvcache
    g = torch.Generator().manual_seed(3)
    codes, scale = torch.zeros(2, 30, 2, 32, 64, dtype=torch.uint8).view(C.F8), torch.zeros(2, 30, 2)
    cuda = codes.cuda(), scale.cuda()
    pos = 0
    for n in (200, 1, 1, 1, 30, 1, 64, 1, 1):
        x = (torch.randn(2, n, 2, 64, generator=g) * 1.7 ** (pos % 40)).bfloat16()
        slots = torch.arange(pos, pos + n, dtype=I32)
        kvcache.append(codes, scale, x[0], x[1], slots)
        kvcache.append(*cuda, x[0].cuda(), x[1].cuda(), slots.cuda())
        pos += n
    clean()
    assert torch.equal(scale, cuda[1].cpu()) and torch.equal(codes.view(torch.uint8), cuda[0].cpu().view(torch.uint8))


def test_append_of_nothing():
    from noeira_b200.ops import kvcache
    kv, scale = torch.zeros(2, 1, 1, 16, 64, dtype=torch.uint8, device="cuda").view(C.F8), torch.zeros(2, 1, 1, device="cuda")
    k = torch.zeros(0, 1, 64, dtype=torch.bfloat16, device="cuda")
    kvcache.append(kv, scale, k, k, torch.zeros(0, dtype=I32, device="cuda"))
    clean()


# ------------------------------------------------------------------------------------------------ attention
def bound(q, d, want, A, c):
    """How far each output may be off; see the head of this file."""
    vals, sc = C.values(d["codes"]), d["scale"].double().numpy()
    kmax = np.nanmax(np.where(np.isnan(vals[0]), 0, np.abs(vals[0])) * sc[0][..., None, None])
    D = q.shape[-1]
    S = c * np.abs(q.float().numpy()).sum(-1).max() * kmax
    n = int(d["ends"].max())
    return 2.0 ** -8 * np.abs(want) + A * (2.0 ** -8 + 2 * (2.0 ** -24 * D * S + 2.0 ** -21) + 2.0 ** -24 * n) + 1e-30


def run_attention(d, max_new="given", out=None, c=None):
    from noeira_b200.ops import kvcache
    q = d["q"].cuda()[: d["T"], 1: 1 + d["hq"]]
    out = torch.full((d["T"] + 3, d["hq"], d["dim"]), 7.0, dtype=torch.bfloat16, device="cuda") if out is None else out
    kvcache.paged_attention(q, d["codes"].cuda(), d["scale"].cuda(), d["tables"].cuda(), d["starts"].cuda(), d["ends"].cuda(),
                            max_new=d["max_new"] if max_new == "given" else max_new, softmax_scale=c, out=out[: d["T"]])
    return out


@pytest.mark.parametrize("case", C.ATTENTION)
def test_attention(case):
    d = C.attention_inputs(case)
    q = d["q"][: d["T"], 1: 1 + d["hq"]]
    c = d["dim"] ** -0.5
    want, A = O.attention(q.float().numpy(), C.values(d["codes"]), d["scale"].double().numpy(), d["tables"].numpy(), d["starts"].numpy(), d["ends"].numpy(), c)
    out = run_attention(d)
    clean()
    err = np.abs(out[: d["T"]].cpu().double().numpy() - want)
    assert np.all(err <= bound(q, d, want, A, c)), (err / bound(q, d, want, A, c)).max()
    assert bool((out[d["T"]:] == 7).all())
    # without the bound of a row's tokens, which changes the launch, not the result's tolerance
    again = run_attention(d, max_new=None)
    clean()
    assert np.all(np.abs(again[: d["T"]].cpu().double().numpy() - want) <= bound(q, d, want, A, c))
    # the same call again gives the same bits
    assert torch.equal(run_attention(d).view(torch.int16), out.view(torch.int16))


def reference(d, q, c):
    """The definition in 64 bits on the GPU, a row at a time: for cases whose loops in Python would take minutes."""
    codes, scale = d["codes"].cuda().double(), d["scale"].cuda().double()
    o, A = torch.zeros(d["T"], d["hq"], d["dim"], dtype=torch.float64, device="cuda"), torch.zeros(d["T"], d["hq"], d["dim"], dtype=torch.float64, device="cuda")
    st, en, G = d["starts"].tolist(), d["ends"].tolist(), d["hq"] // d["hk"]
    for i, end in enumerate(en):
        a, b = st[i], st[i + 1]
        ids = d["tables"][i, : -(-end // d["block"])].long().cuda()
        k, v = ((codes[w, ids] * scale[w, ids][..., None, None]).transpose(0, 1).reshape(d["hk"], -1, d["dim"])[:, :end].repeat_interleave(G, 0) for w in (0, 1))
        see = torch.arange(end, device="cuda")[None] <= (end - (b - torch.arange(a, b, device="cuda")))[:, None]
        p = torch.softmax((q[a:b].cuda().double().transpose(0, 1) @ k.transpose(1, 2) * c).masked_fill(~see, -math.inf), -1)
        o[a:b], A[a:b] = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
    return o.cpu().numpy(), A.cpu().numpy()


@pytest.fixture(params=[0, 1, 2], ids=["by_size", "fragments", "tiles"])
def mode(request):
    """Runs a test once per kernel that rows with many query rows may get."""
    from noeira_b200.ops.kvcache import set_attention_mode
    old = set_attention_mode(request.param)
    yield request.param
    set_attention_mode(old)


@pytest.mark.parametrize("case", C.PROMPTS + C.ATTENTION[7:])
def test_attention_prompts(case, mode):
    d = C.attention_inputs(case)
    q = d["q"][: d["T"], 1: 1 + d["hq"]]
    c = d["dim"] ** -0.5
    want, A = reference(d, q, c)
    out = run_attention(d)
    clean()
    err, most = np.abs(out[: d["T"]].cpu().double().numpy() - want), bound(q, d, want, A, c)
    assert np.all(err <= most), (err / most).max()
    assert bool((out[d["T"]:] == 7).all())
    assert torch.equal(run_attention(d).view(torch.int16), out.view(torch.int16))


def test_attention_prompts_scales_padding_and_a_strided_output(mode):
    """Blocks of very different scales, padded tokens behind the last row, an output whose rows are not 16-byte aligned."""
    from noeira_b200.ops import kvcache
    d = C.attention_inputs(([100, 3], [800, 300], 32, 8, 128, 16), seed=4)
    g = torch.Generator().manual_seed(1)
    d["scale"] = torch.stack([torch.exp2(torch.randint(-9, -5, d["scale"].shape[1:], generator=g).float()), torch.exp2(torch.randint(-14, 6, d["scale"].shape[1:], generator=g).float())])
    T = d["T"] + 77
    q = torch.zeros(T, 32, 128).bfloat16()
    q[: d["T"]] = d["q"][: d["T"], 1:33]
    wide = torch.full((T, 32 * 128 + 2), 7.0, dtype=torch.bfloat16, device="cuda")
    out = wide[:, 1: 1 + 32 * 128].unflatten(1, (32, 128))
    kvcache.paged_attention(q.cuda(), d["codes"].cuda(), d["scale"].cuda(), d["tables"].cuda(), d["starts"].cuda(), d["ends"].cuda(), max_new=800, softmax_scale=0.11, out=out)
    clean()
    assert bool((out[d["T"]:] == 7).all()) and bool((wide[:, 0] == 7).all()) and bool((wide[:, -1] == 7).all())
    want, A = reference(d, q, 0.11)
    assert np.all(np.abs(out[: d["T"]].cpu().double().numpy() - want) <= bound(q, d, want, A, 0.11))


def test_attention_prompts_nan_reaches_only_who_sees_it(mode):
    d = C.attention_inputs(([10, 200], [1300, 700], 16, 16, 64, 32))
    codes = d["codes"].cuda()
    codes.view(torch.uint8)[1, d["tables"][1, 20].item(), 3, 11, 40] = 0xFF      # a value: row 1, place 651, head 3
    codes.view(torch.uint8)[1, d["tables"][1, 3].item(), 3, 11, 41] = 0x7F       # another: place 107, all of the row's tokens see it
    codes.view(torch.uint8)[0, d["tables"][0, 30].item(), 5, 2, 9] = 0x7F        # a key: row 0, place 962, head 5
    d["codes"] = codes
    o = run_attention(d)[: d["T"]]
    clean()
    bad = torch.zeros_like(o, dtype=torch.bool)
    bad[1300 + 651 - 200:, 3, 40] = True
    bad[1300:, 3, 41] = True
    bad[962 - 10: 1300, 5] = True
    assert torch.equal(torch.isnan(o), bad)


def test_attention_prompts_without_keys_and_with_bad_blocks(mode):
    from noeira_b200.ops import check_status
    from noeira_b200.ops.status import DeviceStatusError
    d = C.attention_inputs(([0, 300], [1500, 700], 12, 12, 64, 16))
    d["ends"][0] = 1400                              # the first hundred tokens see nothing
    q = d["q"][: d["T"], 1: 1 + d["hq"]]
    out = run_attention(d)
    clean()
    assert bool((out[:100] == 0).all())
    tail = dict(d, starts=d["starts"].clone(), ends=d["ends"].clone())
    want, A = reference(tail, q, 0.125)
    keep = slice(100, d["T"])
    assert np.all(np.abs(out[keep].cpu().double().numpy() - want[keep]) <= bound(q, d, want[keep], A[keep], 0.125))
    for bad in (-1, 1 << 30):
        e = dict(d, tables=d["tables"].clone())
        e["tables"][0, 40] = bad
        again = run_attention(e)
        with pytest.raises(DeviceStatusError, match="bounds"):
            check_status()
        assert torch.equal(again[1500: d["T"]], out[1500: d["T"]])


@pytest.mark.parametrize("case", [C.ATTENTION[3], C.ATTENTION[8], C.ATTENTION[10]])
def test_attention_scales_of_any_size(case):
    """Blocks whose scales differ by 2^20, scores far from zero, another softmax scale."""
    d = C.attention_inputs(case, seed=9)
    g = torch.Generator().manual_seed(1)
    d["scale"] = torch.stack([torch.exp2(torch.randint(-9, -3, d["scale"].shape[1:], generator=g).float()), torch.exp2(torch.randint(-14, 6, d["scale"].shape[1:], generator=g).float())])
    q = d["q"][: d["T"], 1: 1 + d["hq"]]
    want, A = O.attention(q.float().numpy(), C.values(d["codes"]), d["scale"].double().numpy(), d["tables"].numpy(), d["starts"].numpy(), d["ends"].numpy(), 0.31)
    out = run_attention(d, c=0.31)
    clean()
    assert np.all(np.abs(out[: d["T"]].cpu().double().numpy() - want) <= bound(q, d, want, A, 0.31))


@pytest.mark.parametrize("new", [1, 40, 200])
def test_attention_padded_tokens_are_left(new):
    """Tokens behind the last row's keep what ``out`` held, also inside the last tile."""
    from noeira_b200.ops import kvcache
    d = C.attention_inputs(([70, 3], [new, 1], 4, 2, 64, 32))
    T = d["T"] + 37
    q = torch.randn(T, 4, 64, device="cuda").bfloat16()
    out = torch.full_like(q, 7)
    kvcache.paged_attention(q, d["codes"].cuda(), d["scale"].cuda(), d["tables"].cuda(), d["starts"].cuda(), d["ends"].cuda(), max_new=new, out=out)
    clean()
    assert bool((out[d["T"]:] == 7).all()) and bool(torch.isfinite(out).all())
    want, A = O.attention(q[: d["T"]].cpu().float().numpy(), C.values(d["codes"]), d["scale"].double().numpy(), d["tables"].numpy(), d["starts"].numpy(), d["ends"].numpy(), 0.125)
    assert np.all(np.abs(out[: d["T"]].cpu().double().numpy() - want) <= bound(q.cpu(), d, want, A, 0.125))


@pytest.mark.parametrize("tokens", [2, 40, 140])
def test_attention_token_that_sees_nothing_is_zero(tokens):
    from noeira_b200.ops import kvcache
    kv, scale = C.random_codes((2, 12, 2, 16, 64), 1, nan=True).cuda(), torch.ones(2, 12, 2, device="cuda")
    q = torch.randn(tokens, 4, 64, device="cuda").bfloat16()
    # the row holds one token fewer than the call's: its first token sees nothing; a second row is empty
    t = torch.arange(12, dtype=I32, device="cuda").reshape(1, 12).repeat(2, 1)
    kv.view(torch.uint8)[:, :, :, :, :] = C.random_codes((2, 12, 2, 16, 64), 2).view(torch.uint8).cuda()
    o = kvcache.paged_attention(q, kv, scale, t, ints([0, tokens - 1, tokens]), ints([tokens - 2, 0]), max_new=tokens)
    clean()
    assert bool((o[0] == 0).all()) and bool((o[-1] == 0).all())
    if tokens > 2:
        assert bool((o[1:-1] != 0).any(-1).all())


@pytest.mark.parametrize("tokens", [1, 30, 140])
def test_attention_nan_in_the_cache_reaches_only_who_sees_it(tokens):
    from noeira_b200.ops import kvcache
    case = ([50, 90], [tokens, tokens], 4, 2, 64, 16)
    d = C.attention_inputs(case)
    codes = d["codes"].cuda()
    codes.view(torch.uint8)[1, d["tables"][1, 2].item(), 1, 3, 5] = 0x7F         # a value: row 1, place 35, head 1, dimension 5
    d["codes"] = codes
    o = run_attention(d)[: d["T"]]
    clean()
    bad = torch.zeros_like(o, dtype=torch.bool)
    bad[tokens:, 2:, 5] = True
    assert torch.equal(torch.isnan(o), bad)
    d["codes"].view(torch.uint8)[0, d["tables"][0, 0].item(), 0, 0, 9] = 0x7F    # a key: row 0, place 0, head 0
    o = run_attention(d)[: d["T"]]
    clean()
    bad[:tokens, :2] = True
    assert torch.equal(torch.isnan(o), bad)


@pytest.mark.parametrize("tokens", [1, 20, 150])
@pytest.mark.parametrize("bad", [-1, 1000, 0x7fffffff])
def test_attention_bad_block_id_is_reported(tokens, bad):
    from noeira_b200.ops import check_status
    from noeira_b200.ops.status import DeviceStatusError
    d = C.attention_inputs(([200, 90], [tokens, 1], 4, 2, 64, 16))
    d["tables"][0, 4] = bad
    want, A = O.attention(d["q"][: d["T"], 1:5].float().numpy(), C.values(d["codes"]), d["scale"].double().numpy(), d["tables"].numpy(), d["starts"].numpy(), d["ends"].numpy(), 0.125, skip=(0,))
    out = run_attention(d)
    with pytest.raises(DeviceStatusError, match="bounds"):
        check_status()
    last = slice(tokens, tokens + 1)                                             # the other row is not touched by it
    assert np.all(np.abs(out[last].cpu().double().numpy() - want[last]) <= bound(d["q"], d, want[last], A[last], 0.125))


def test_attention_offsets_past_32_bits():
    """A cache layer of more than 2^32 bytes, the row's blocks at its end."""
    from noeira_b200.ops import kvcache
    heads, block, dim = 8, 128, 128
    blocks = (1 << 32) // (heads * block * dim) + 3
    kv = torch.empty(2, blocks, heads, block, dim, dtype=torch.uint8, device="cuda").view(C.F8)
    scale = torch.ones(2, blocks, heads, device="cuda")
    t = ints([[blocks - 1, 0, blocks - 2]])
    small = C.random_codes((2, 3, heads, block, dim), 3)
    sc = torch.exp2(torch.randint(-9, -6, (2, 3, heads)).float())
    for i, b in enumerate(t[0].tolist()):
        kv.view(torch.uint8)[:, b] = small.view(torch.uint8)[:, i].cuda()
        scale[:, b] = sc[:, i].cuda()
    for n in (1, 150):
        q = torch.randn(n, 16, dim, device="cuda").bfloat16()
        a = kvcache.paged_attention(q, kv, scale, t, ints([0, n]), ints([300]), max_new=n)
        b = kvcache.paged_attention(q, small.cuda(), sc.cuda(), ints([[0, 1, 2]]), ints([0, n]), ints([300]), max_new=n)
        clean()
        assert torch.equal(a, b)
    x = torch.randn(2, 2, heads, dim, device="cuda").bfloat16()
    slots = ints([(blocks - 2) * block + 44, (blocks - 2) * block + 45])
    kvcache.append(kv, scale, x[0], x[1], slots)
    two, tsc = small.cuda(), sc.cuda()
    kvcache.append(two, tsc, x[0], x[1], ints([2 * block + 44, 2 * block + 45]))
    clean()
    assert torch.equal(kv[:, blocks - 2, :, :46].view(torch.uint8), two[:, 2, :, :46].view(torch.uint8)) and torch.equal(scale[:, blocks - 2], tsc[:, 2])


def test_attention_two_streams_and_a_captured_graph():
    """Calls on two streams at once and a replayed graph beside eager calls give the same bits as one call alone."""
    from noeira_b200.ops import kvcache
    cases = [C.attention_inputs(([3000, 17, 900], [1, 1, 1], 8, 2, 64, 16), 1), C.attention_inputs(([800, 1500, 20], [1, 130, 3], 8, 2, 64, 16), 2)]
    args = []
    for d in cases:
        q = d["q"].cuda()[: d["T"], 1: 1 + d["hq"]].contiguous()
        args.append((q, d["codes"].cuda(), d["scale"].cuda(), d["tables"].cuda(), d["starts"].cuda(), d["ends"].cuda(), d["max_new"]))
    want = [kvcache.paged_attention(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    outs, graphs = [[] for _ in args], []
    for a, s in zip(args, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            o = kvcache.paged_attention(*a)
        graphs.append((g, o))
    for _ in range(20):
        for i, (a, s) in enumerate(zip(args, streams)):
            with torch.cuda.stream(s):
                outs[i].append(kvcache.paged_attention(*a))
                graphs[i][0].replay()
    clean()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i]) and torch.equal(graphs[i][1], want[i])


# ------------------------------------------------------------------------------------------------ beams
def check_select(x, scores, fin, eos, got):
    """Tokens and parents equal the definition's; where two values are nearer than fp32 sums can tell, either order is right."""
    s, p, t, done = (v.cpu() for v in got)
    beams = s.shape[1]
    for r, row in enumerate(O.select(x, scores, fin, eos)):
        assert [(int(a), int(b)) for a, b in zip(p[r], t[r])] == [(b, v) for _, b, v in row], r
        vals = np.array([v for v, _, _ in row])
        top = np.nan_to_num(np.abs(scores[r].cpu().double().numpy()), nan=0, posinf=0).max() + 40
        assert np.array_equal(np.isinf(s[r].numpy()), np.isinf(vals))
        fine = np.isfinite(vals)
        # fp32 sum of exponentials of 2^-22 each, log; the value itself rounds to 2^-24
        assert np.all(np.abs(s[r].double().numpy()[fine] - vals[fine]) <= 2.0 ** -20 + 2.0 ** -24 * top)
        for k in range(beams):
            assert bool(done[r, k]) == (eos is not None and ((fin is not None and bool(fin[r, p[r, k]])) or int(t[r, k]) == eos))


@pytest.mark.parametrize("requests,beams,vocab", [(1, 1, 1), (1, 4, 49152), (3, 8, 1000), (2, 5, 32003), (2, 32, 4099), (70, 2, 257), (1, 3, 2), (2, 16, 9), (1, 31, 8193), (4, 12, 65000)])
@pytest.mark.parametrize("fp32", [False, True])
def test_select(requests, beams, vocab, fp32):
    from noeira_b200.ops import beam
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(requests, beams, vocab, generator=g) * 3
    x = x if fp32 else x.bfloat16()
    scores = -torch.rand(requests, beams, generator=g) * 10
    check_select(x, scores, None, None, beam.beam_select(x.cuda(), scores.cuda()))
    fin = torch.rand(requests, beams, generator=g) < 0.3
    scores[:, beams // 2 + 1:] = -math.inf
    eos = vocab // 2
    check_select(x, scores, fin, eos, beam.beam_select(x.cuda(), scores.cuda(), finished=fin.cuda(), eos=eos))
    check_select(x, scores, None, eos, beam.beam_select(x.cuda(), scores.cuda(), eos=eos))


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "few", "nan", "none", "inf", "blocks"])
def test_select_orders_and_ties(kind, fp32):
    from noeira_b200.ops import beam
    R, B, V = 2, 8, 20011
    v = torch.arange(V).float()
    x = {"equal": torch.zeros(V), "rising": v / 64, "falling": -v / 64, "few": torch.full((V,), -math.inf), "nan": torch.full((V,), math.nan), "none": torch.full((V,), -math.inf), "inf": v * 0,
         "blocks": (v // 4000) % 2}[kind].expand(R, B, V).clone()
    if kind == "few":
        x[:, 0, 17000], x[:, 3, 5], x[0, 3, 20010] = 1.0, 2.0, 2.0
    if kind == "nan":
        x[:, 1, 777] = -3.0
    if kind == "inf":
        x[:, 2, 400], x[:, 2, 19000], x[:, 4, 3] = math.inf, math.inf, -math.inf
    x = x if fp32 else x.bfloat16()
    scores = torch.tensor([[0.0] * B, [-1.0, -1.0, 0.0, -math.inf, 0.0, math.nan, -2.0, 0.0]])
    check_select(x, scores, None, None, beam.beam_select(x.cuda(), scores.cuda()))


def test_select_padded_rows():
    from noeira_b200.ops import beam
    g = torch.Generator().manual_seed(0)
    for pitch in (1008, 1001):
        wide = torch.randn(3, 4, pitch, generator=g).bfloat16()
        wide[..., 1000:] = 50                                # what lies between the rows is not looked at
        scores = -torch.rand(3, 4, generator=g)
        check_select(wide[..., :1000], scores, None, None, beam.beam_select(wide.cuda()[..., :1000], scores.cuda()))


@pytest.mark.parametrize("beams,heads,dim,block,layers", [(2, 1, 64, 16, 1), (4, 6, 64, 16, 6), (8, 5, 128, 64, 3), (3, 2, 64, 128, 2)])
def test_reorder(beams, heads, dim, block, layers):
    from noeira_b200.ops import beam
    rng = np.random.RandomState(beams)
    lens = [n for n in (1, block, block * 3 - 1, 2 * block + 5) for _ in range(beams)]
    tables, blocks, left = C.paged(lens, block, 2, spare_blocks=len(lens))
    codes = C.random_codes((layers, 2, blocks, heads, block, dim), 4)
    scale = torch.rand(layers, 2, blocks, heads)
    parents = rng.randint(0, beams, (4, beams)).astype(np.int32)
    parents[1] = np.arange(beams)
    want = O.reorder(C.values(codes), scale.numpy(), tables, lens, parents, left)
    c, sc = codes.cuda(), scale.cuda()
    for _ in range(2):                                       # a second call on the same inputs writes the same
        t, n, s = beam.beam_reorder(c, sc, torch.from_numpy(tables).cuda(), ints(lens), torch.from_numpy(parents).cuda(), ints(left.tolist()))
        clean()
        for a, b in zip((C.values(c), sc.cpu().numpy(), t.cpu().numpy(), n.cpu().numpy(), s.cpu().numpy()), want):
            assert np.array_equal(a, b)


def test_reorder_reports_bad_parents_and_missing_blocks():
    from noeira_b200.ops import beam, check_status
    from noeira_b200.ops.status import DeviceStatusError
    codes = C.random_codes((1, 2, 6, 1, 16, 64), 4).cuda()
    scale = torch.ones(1, 2, 6, 1, device="cuda")
    before = codes.clone()
    for parents, spare, tables in (([[5, 1]], [2, 3], [[0], [1]]), ([[-1, 1]], [2, 3], [[0], [1]]), ([[1, 1]], [-1, 3], [[0], [1]]), ([[1, 1]], [6, 3], [[0], [1]]), ([[1, 1]], [2, 3], [[0], [77]])):
        beam.beam_reorder(codes, scale, ints(tables), ints([3, 3]), ints(parents), ints(spare))
        with pytest.raises(DeviceStatusError, match="bounds"):
            check_status()
        assert torch.equal(codes.view(torch.uint8), before.view(torch.uint8))


# ------------------------------------------------------------------------------------------------ together
def test_cache_through_prompts_steps_and_reorders():
    """A run as a decoder makes it: prompts, a fan-out to beams, steps with reorders; the cache stays what the CPU form gives,
    and attention over it what the definition gives."""
    from noeira_b200.ops import kvcache
    g = torch.Generator().manual_seed(5)
    heads, hq, dim, layers, beams = 2, 4, 64, 2, 3
    caches = [kvcache.PagedKVCache(layers, heads, dim, blocks=60, rows=2 * beams, max_len=90, block=16, device=dev, spares=True) for dev in ("cpu", "cuda")]
    first = [0] * (2 * beams)
    first[0], first[beams] = 37, 16
    steps = [first] + [[1] * (2 * beams)] * 30
    for n, new in enumerate(steps):
        T = sum(new)
        x = torch.randn(layers, T, hq + 2 * heads, dim, generator=g).bfloat16()
        outs = []
        for c in caches:
            p = c.plan(torch.tensor(new, dtype=I32, device=c.device), T)
            xs = x.to(c.device)
            for l in range(layers):
                c.append(l, xs[l][:, hq: hq + heads], xs[l][:, hq + heads:], p)
            outs.append(torch.stack([c.attend(l, xs[l][:, :hq], p, max_new=max(new)).float().cpu() for l in range(layers)]))
        a, b = caches
        assert torch.equal(a.tables, b.tables.cpu()) and torch.equal(a.lengths, b.lengths.cpu()) and torch.equal(a.spare, b.spare.cpu()) and int(a.free_count) == int(b.free_count)
        assert torch.equal(a.scale, b.scale.cpu()) and torch.equal(a.kv.view(torch.uint8), b.kv.cpu().view(torch.uint8))
        # bf16 output and weights, |v| at most 6 of these normal draws
        assert float((outs[0] - outs[1]).abs().max()) <= 2 * 2.0 ** -8 * 6
        parents = torch.zeros(2, beams, dtype=I32) if n == 0 else torch.randint(0, beams, (2, beams), generator=g).to(I32)
        for c in caches:
            c.reorder(parents.to(c.device))
            if n == 0:
                c.refill_spares()
    clean()
    for c in caches:
        c.reset([0, 1, 2])
    assert int(caches[0].free_count) == int(caches[1].free_count)


def test_attention_prompts_in_a_batch_of_many_rows():
    """More rows than a block has threads: single tokens, rows without new ones and a few prompts among them."""
    n = 500
    held = [(7 * i) % 23 for i in range(n)]
    new = [1 if i % 3 else 0 for i in range(n)]
    new[0], new[250], new[499], held[250] = 700, 900, 1000, 300
    d = C.attention_inputs((held, new, 12, 12, 64, 16))
    q = d["q"][: d["T"], 1:13]
    want, A = reference(d, q, 0.125)
    out = run_attention(d)
    clean()
    assert np.all(np.abs(out[: d["T"]].cpu().double().numpy() - want) <= bound(q, d, want, A, 0.125))


@pytest.mark.parametrize("case", [C.ATTENTION[3], C.ATTENTION[7], C.ATTENTION[12], C.PROMPTS[1], C.PROMPTS[3]])
def test_attention_queries_on_odd_addresses(case, mode):
    """Query rows that begin on no 16-byte boundary, as views of a wider matrix, give the bits of aligned ones."""
    from noeira_b200.ops import kvcache
    d = C.attention_inputs(case)
    T, hq, dim = d["T"], d["hq"], d["dim"]
    q = d["q"][:T, 1: 1 + hq].contiguous().cuda()
    wide = torch.zeros(T, hq * dim + 3, dtype=torch.bfloat16, device="cuda")
    odd = wide[:, 1: 1 + hq * dim].unflatten(1, (hq, dim))
    odd.copy_(q)
    rest = (d["codes"].cuda(), d["scale"].cuda(), d["tables"].cuda(), d["starts"].cuda(), d["ends"].cuda(), d["max_new"])
    a, b = kvcache.paged_attention(q, *rest), kvcache.paged_attention(odd, *rest)
    clean()
    assert torch.equal(a, b)


def test_plan_in_a_captured_graph_counts_down():
    """A plan of many tokens, captured with its counter in place: each replay takes the next blocks."""
    from noeira_b200.ops import kvcache
    rows, new, width = 40, 20, 12
    tables = torch.full((rows, width), -1, dtype=I32, device="cuda")
    lengths, free, count = torch.zeros(rows, dtype=I32, device="cuda"), torch.arange(rows * width, dtype=I32, device="cuda"), ints([rows * width])
    add = torch.full((rows,), new, dtype=I32, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        p = kvcache.plan_tokens(tables, lengths, add, free, count, 16, rows * new)
        lengths.copy_(p.ends)
    left = rows * width
    for n in range(1, 9):
        g.replay()
        torch.cuda.synchronize()
        left -= rows * (-(-n * new // 16) + -(n - 1) * new // 16)
        used = tables[tables >= 0]
        assert int(count) == left and bool((lengths == n * new).all()) and used.numel() == rows * width - left == used.unique().numel()
    clean()
