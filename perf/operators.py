"""Serving a decoder language model from a paged key / value cache held in 8 bits: the operators, their cases, plain forms and
64-bit results.

  plan     block tables and slot maps from the lengths of the requests (``ops.kvcache.plan_tokens``)
  append   new keys and values into the cache, one power-of-two scale per block and head (``ops.kvcache.append``)
  attend   causal attention of new tokens over the cache: prompts, chunks of prompts, single tokens (``ops.kvcache.paged_attention``)
  select   the best continuations over beams and vocabulary (``ops.beam.beam_select``)
  reorder  the cache's tables and partly filled blocks follow the selected beams (``ops.beam.beam_reorder``)

Layouts: codes e4m3 ``[2, blocks, heads, block, head_dim]`` (keys, values; a leading layer dimension for ``reorder``), scales fp32
``[2, blocks, heads]``, tables int32 ``[rows, width]``.  The tokens of a call are ragged: row i owns ``starts[i] .. starts[i + 1]``.
"""
import math

import torch

own = False

DEV = "cuda"
F8 = torch.float8_e4m3fn
TOP = 448.0             # largest e4m3 value
LEAST = -118            # exponent of the smallest scale


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of a small server: 64 requests get a token each, four of 64 cross into a new block
        dict(name="plan_step", op="plan", rows=64, len_lo=5, len_hi=1000, new_lo=1, new_hi=1, block=16),
        # admission of a large batch of prompts of very different lengths
        dict(name="plan_prompts", op="plan", rows=2048, len_lo=0, len_hi=700, new_lo=1, new_hi=2048, block=16),
        # the new token of each request in a decode step, heads of the vision-language model's decoder
        dict(name="append_step", op="append", rows=64, len_lo=5, len_hi=1000, new_lo=1, new_hi=1, heads=5, dim=64, block=16),
        # prompts going into an empty or partly filled cache
        dict(name="append_prompts", op="append", rows=24, len_lo=0, len_hi=333, new_lo=100, new_hi=4096, heads=8, dim=128, block=32),
        # one user, one token: the default GPT's heads, latency counts
        dict(name="attend_one_token", op="attend", rows=1, len_lo=639, len_hi=639, new_lo=1, new_hi=1, q_heads=6, heads=6, dim=64, block=16),
        # a decode step of a server: ragged lengths, three query heads to a key head
        dict(name="attend_tokens", op="attend", rows=96, len_lo=32, len_hi=4096, new_lo=1, new_hi=1, q_heads=15, heads=5, dim=64, block=16),
        # few requests with very long caches
        dict(name="attend_tokens_long", op="attend", rows=8, len_lo=16384, len_hi=65535, new_lo=1, new_hi=1, q_heads=32, heads=8, dim=128, block=64),
        # chunks of prompts over what the cache holds of them already
        dict(name="attend_prompts", op="attend", rows=4, len_lo=0, len_hi=4000, new_lo=700, new_hi=2048, q_heads=32, heads=8, dim=128, block=32),
        # beam search for one user over the decoder's vocabulary
        dict(name="select_one", op="select", requests=1, beams=4, vocab=49152, dtype="bf16", finished=False),
        # a batch of searches over an odd vocabulary in fp32, some beams finished
        dict(name="select_many", op="select", requests=48, beams=8, vocab=32003, dtype="fp32", finished=True),
        # the cache of one search of the default GPT
        dict(name="reorder_one", op="reorder", requests=1, beams=4, layers=6, heads=6, dim=64, block=16, len_lo=300, len_hi=300),
        # the caches of a batch of searches, 16 layers
        dict(name="reorder_many", op="reorder", requests=48, beams=8, layers=16, heads=5, dim=64, block=64, len_lo=40, len_hi=1500),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(max(lo, 0.5)), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("plan", "append", "attend", "attend", "attend", "select", "reorder"))
    block = rng.choice((16, 32, 64, 128))
    dim = rng.choice((64, 128))
    if op == "plan":
        lo = _log(rng, 1, 64)
        c = dict(op=op, rows=_log(rng, 1, 2048), len_lo=0, len_hi=_log(rng, 1, 4000), new_lo=lo, new_hi=_log(rng, lo, 2048), block=block)
    elif op == "append":
        lo = _log(rng, 1, 512)
        c = dict(op=op, rows=_log(rng, 1, 128), len_lo=rng.randint(0, 70), len_hi=_log(rng, 71, 3000), new_lo=lo, new_hi=_log(rng, lo, 4096), heads=rng.choice((1, 2, 4, 5, 6, 8, 15)),
                 dim=dim, block=block)
    elif op == "attend":
        heads, group = rng.choice(((6, 1), (5, 3), (2, 8), (8, 4), (1, 16), (3, 2), (12, 1)))
        kind = rng.choice(("tokens", "chunks", "prompts", "mixed"))
        c = dict(op=op, q_heads=heads * group, heads=heads, dim=dim, block=block)
        if kind == "tokens":
            c.update(rows=_log(rng, 1, 256), len_lo=rng.randint(0, 900), len_hi=_log(rng, 901, 40000), new_lo=1, new_hi=1)
        elif kind == "chunks":      # a few tokens at once: a draft that is checked, the last piece of a prompt
            c.update(rows=_log(rng, 1, 64), len_lo=rng.randint(0, 300), len_hi=_log(rng, 301, 8000), new_lo=2, new_hi=rng.randint(2, 40))
        elif kind == "prompts":
            c.update(rows=rng.randint(1, 6), len_lo=0, len_hi=_log(rng, 1, 4000), new_lo=_log(rng, 64, 900), new_hi=_log(rng, 900, 2048))
        else:                       # prompts and single tokens in one call
            c.update(rows=rng.randint(4, 24), len_lo=rng.randint(0, 100), len_hi=_log(rng, 200, 4000), new_lo=1, new_hi=_log(rng, 100, 1000))
    elif op == "select":
        c = dict(op=op, requests=_log(rng, 1, 64), beams=rng.randint(1, 16), vocab=_log(rng, 50, 65000), dtype=rng.choice(("bf16", "fp32")), finished=rng.random() < 0.5)
    else:
        c = dict(op=op, requests=_log(rng, 1, 48), beams=rng.randint(2, 12), layers=rng.randint(1, 16), heads=rng.choice((1, 5, 6, 8)), dim=dim, block=block, len_lo=rng.randint(1, 60),
                 len_hi=_log(rng, 61, 1500))
    cap = {"plan": 8e6, "append": 1.6e8, "attend": 5.8e8, "select": 4.9e7, "reorder": 2.0e8}[op]
    rows = "requests" if "requests" in c else "rows"
    while c[rows] > 1 and (work(c)["bytes"] > cap or work(c)["flops"] > 2.0e11 or _held(c) > 3e9):
        c[rows] = (c[rows] + 1) // 2
    return c


def _held(c):
    """Bytes of cache that the state of a case holds."""
    if c["op"] == "reorder":
        return c["layers"] * _reorder_blocks(c) * 2 * c["heads"] * c["block"] * c["dim"]
    if c["op"] in ("append", "attend"):
        return 2 * _blocks(c) * c["heads"] * c["block"] * c["dim"]
    return 0


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, spread evenly over the logarithm: what the case alone fixes; the seed only orders them."""
    if n == 1 or lo == hi:
        return [hi] * n
    a, b = math.log(lo + 1), math.log(hi + 1)
    return [min(hi, max(lo, int(round(math.exp(a + (b - a) * i / (n - 1)))) - 1)) for i in range(n)]


def _lengths(c):
    """Tokens held and tokens new of each row, in the case's own order (the pairing is fixed: long and short prompts mix)."""
    held, new = _spread(c["rows"], c["len_lo"], c["len_hi"]), _spread(c["rows"], c["new_lo"], c["new_hi"])
    step = next(s for s in range(max(1, int(c["rows"] * 0.618)), c["rows"] + 1) if math.gcd(s, c["rows"]) == 1 or c["rows"] == 1)
    return held, [new[(i * step) % c["rows"]] for i in range(c["rows"])]


def _need(tokens, block):
    return -(-tokens // block)


def _blocks(c):
    held, new = _lengths(c)
    return sum(_need(h + n, c["block"]) for h, n in zip(held, new)) + 3


def _reorder_blocks(c):
    return sum(c["beams"] * (_need(n, c["block"]) + 1) for n in _spread(c["requests"], c["len_lo"], c["len_hi"])) + 3


def work(case):
    c, op = case, case["op"]
    if op == "select":
        rows = c["requests"] * c["beams"]
        return {"bytes": rows * (c["vocab"] * (2 if c["dtype"] == "bf16" else 4) + 4 + 12 + 2), "flops": 4.0 * rows * c["vocab"]}
    if op == "reorder":
        # about half of the beams have another parent; in a step every one of them may, which is what the case does
        part = sum(n % c["block"] for n in _spread(c["requests"], c["len_lo"], c["len_hi"])) * (c["beams"] - 1)
        tables = sum(_need(n, c["block"]) for n in _spread(c["requests"], c["len_lo"], c["len_hi"])) * c["beams"]
        return {"bytes": 2.0 * part * c["layers"] * 2 * c["heads"] * c["dim"] + 8.0 * tables, "flops": 0.0}
    held, new = _lengths(c)
    tokens = sum(new)
    if op == "plan":
        fresh = sum(_need(h + n, c["block"]) - _need(h, c["block"]) for h, n in zip(held, new))
        return {"bytes": c["rows"] * 20.0 + 8.0 * fresh + 12.0 * tokens, "flops": 0.0}
    if op == "append":
        return {"bytes": 6.0 * tokens * c["heads"] * c["dim"] + 4.0 * tokens, "flops": 0.0}
    seen = sum(h + n for h, n in zip(held, new))
    pairs = sum(n * h + n * (n + 1) // 2 for h, n in zip(held, new))
    return {"bytes": 2.0 * seen * c["heads"] * c["dim"] + 4.0 * tokens * c["q_heads"] * c["dim"], "flops": 4.0 * pairs * c["q_heads"] * c["dim"]}


# ------------------------------------------------------------------------------------------------ inputs
class State:
    pass


def _ints(v, gen=None):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _codes(shape, gen):
    """Codes of normally distributed values, as a cache holds them."""
    out = torch.empty(shape, dtype=F8, device=DEV)
    flat = out.view(torch.uint8).reshape(-1)
    for at in range(0, flat.numel(), 1 << 27):
        n = min(1 << 27, flat.numel() - at)
        flat[at: at + n] = (torch.randn(n, device=DEV, generator=gen) * 70).clamp_(-TOP, TOP).to(F8).view(torch.uint8)
    return out


def _scales(shape, gen):
    return ((torch.randint(-9, -5, shape, device=DEV, generator=gen, dtype=torch.int32) + 127) << 23).view(torch.float32)


def _rows(c, gen):
    """Lengths in the order of the seed, tables over shuffled blocks with room for the new tokens."""
    s = State()
    held, new = _lengths(c)
    order = torch.randperm(c["rows"], device=DEV, generator=gen).tolist()
    held, new = [held[i] for i in order], [new[i] for i in order]
    s.held, s.new = held, new
    s.block = c["block"]
    s.lengths, s.new_lens = _ints(held), _ints(new)
    s.blocks = _blocks(c)
    s.width = max(_need(h + n, c["block"]) for h, n in zip(held, new)) + 1
    s.ids = torch.randperm(s.blocks, device=DEV, generator=gen).to(torch.int32)
    return s


def _tables(s, filled):
    """Tables whose first ``filled[i]`` entries are taken off the shuffled ids in turn; returns how many were taken."""
    n = torch.tensor(filled, device=DEV)
    off = n.cumsum(0) - n
    col = torch.arange(s.width, device=DEV)[None]
    at = (off[:, None] + col).clamp_max(s.blocks - 1)
    s.tables = torch.where(col < n[:, None], s.ids[at], torch.full_like(at, -1, dtype=torch.int32)).to(torch.int32)
    return sum(filled)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(1000 + seed)
    if c["op"] == "select":
        s = State()
        s.op, s.beams, s.eos = "select", c["beams"], 2 if c["finished"] else None
        x = torch.randn(c["requests"], c["beams"], c["vocab"], device=DEV, generator=gen) * 3
        s.logits = x.to(torch.bfloat16 if c["dtype"] == "bf16" else torch.float32)
        s.scores = -torch.rand(c["requests"], c["beams"], device=DEV, generator=gen) * 20
        s.finished = (torch.rand(c["requests"], c["beams"], device=DEV, generator=gen) < 0.2) if c["finished"] else None
        return s
    if c["op"] == "reorder":
        s = State()
        s.op, s.block, s.beams = "reorder", c["block"], c["beams"]
        per = _spread(c["requests"], c["len_lo"], c["len_hi"])
        order = torch.randperm(c["requests"], device=DEV, generator=gen).tolist()
        lens = [per[i] for i in order for _ in range(c["beams"])]
        s.held = lens
        s.blocks = _reorder_blocks(c)
        s.width = max(_need(n, c["block"]) for n in lens) + 1
        s.ids = torch.randperm(s.blocks, device=DEV, generator=gen).to(torch.int32)
        used = _tables(s, [_need(n, c["block"]) for n in lens])
        s.spare = s.ids[used: used + len(lens)].contiguous()
        s.lengths = _ints(lens)
        s.kv = _codes((c["layers"], 2, s.blocks, c["heads"], c["block"], c["dim"]), gen)
        s.scale = _scales((c["layers"], 2, s.blocks, c["heads"]), gen)
        # every beam follows another one
        shift = torch.randint(1, c["beams"], (c["requests"], c["beams"]), device=DEV, generator=gen)
        s.parents = ((torch.arange(c["beams"], device=DEV)[None] + shift) % c["beams"]).to(torch.int32)
        s.tables_out, s.lengths_out, s.spare_out = torch.empty_like(s.tables), torch.empty_like(s.lengths), torch.empty_like(s.spare)
        return s
    s = _rows(c, gen)
    s.op = c["op"]
    s.tokens = sum(s.new)
    if c["op"] == "plan":
        used = _tables(s, [_need(h, c["block"]) for h in s.held])
        s.free = s.ids[used:].contiguous()
        s.free_count, s.free_count_out = _ints([s.free.numel()]), _ints([0])
        return s
    _tables(s, [_need(h + n, c["block"]) for h, n in zip(s.held, s.new)])
    s.starts = torch.cat([torch.zeros(1, dtype=torch.int32, device=DEV), s.new_lens.cumsum(0).to(torch.int32)])
    s.ends = s.lengths + s.new_lens
    s.max_new = max(s.new)
    s.kv = _codes((2, s.blocks, c["heads"], c["block"], c["dim"]), gen)
    s.scale = _scales((2, s.blocks, c["heads"]), gen)
    if c["op"] == "attend":
        s.q = (torch.randn(s.tokens, c["q_heads"], c["dim"], device=DEV, generator=gen) * 2).to(torch.bfloat16)
        s.out = torch.empty_like(s.q)
        return s
    # the projection's packed output: keys and values are views of one matrix, with a few larger channels
    qkv = torch.randn(s.tokens, 3 * c["heads"], c["dim"], device=DEV, generator=gen) * (1 + 7 * (torch.rand(3 * c["heads"], c["dim"], device=DEV, generator=gen) < 0.03))
    s.qkv = qkv.to(torch.bfloat16)
    s.k, s.v = s.qkv[:, c["heads"]: 2 * c["heads"]], s.qkv[:, 2 * c["heads"]:]
    row = torch.repeat_interleave(torch.arange(c["rows"], device=DEV), s.new_lens, output_size=s.tokens)
    pos = s.lengths[row] + torch.arange(s.tokens, device=DEV, dtype=torch.int32) - s.starts[row]
    s.slots = (s.tables[row, (pos // c["block"]).long()] * c["block"] + pos % c["block"]).to(torch.int32)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    s = state
    if own:
        from noeira_b200.ops import beam, kvcache
        if s.op == "plan":
            p = kvcache.plan_tokens(s.tables, s.lengths, s.new_lens, s.free, s.free_count, s.block, s.tokens, free_count_out=s.free_count_out)
            return {"tables": s.tables, "starts": p.starts, "ends": p.ends, "rows": p.rows, "positions": p.positions, "slots": p.slots, "free_count": p.free_count}
        if s.op == "append":
            kvcache.append(s.kv, s.scale, s.k, s.v, s.slots)
            return {"kv": s.kv, "scale": s.scale}
        if s.op == "attend":
            return kvcache.paged_attention(s.q, s.kv, s.scale, s.tables, s.starts, s.ends, max_new=s.max_new, out=s.out)
        if s.op == "select":
            return beam.beam_select(s.logits, s.scores, finished=s.finished, eos=s.eos)
        beam.beam_reorder(s.kv, s.scale, s.tables, s.lengths, s.parents, s.spare, tables_out=s.tables_out, lengths_out=s.lengths_out, spare_out=s.spare_out)
        return {"kv": s.kv, "scale": s.scale, "tables": s.tables_out, "lengths": s.lengths_out, "spare": s.spare_out}
    return {"plan": _plan, "append": _append, "attend": _attend, "select": _select, "reorder": _reorder}[s.op](s)


def _plan(s):
    n, b = s.lengths.numel(), s.block
    have = (s.lengths + (b - 1)) // b
    end = s.lengths + s.new_lens
    need = (end + (b - 1)) // b - have
    starts = torch.zeros(n + 1, dtype=torch.int32, device=DEV)
    starts[1:] = s.new_lens.cumsum(0)
    fits = (end <= s.tables.shape[1] * b) & (starts[1:] <= s.tokens)
    need = torch.where(fits, need, torch.zeros_like(need))
    upto = need.cumsum(0).to(torch.int32)
    off = upto - need
    granted = fits & ((need == 0) | (upto <= s.free_count))
    col = torch.arange(s.tables.shape[1], device=DEV, dtype=torch.int32)[None]
    k = col - have[:, None]
    fresh = granted[:, None] & (k >= 0) & (k < need[:, None])
    at = (s.free_count - 1 - off[:, None] - k).clamp(0, s.free.numel() - 1)
    s.tables.copy_(torch.where(fresh, s.free[at.long()], s.tables))
    t = torch.arange(s.tokens, device=DEV, dtype=torch.int32)
    row = torch.searchsorted(starts[1:], t, right=True)
    behind = row >= n
    row = row.clamp_max(n - 1)
    pos = s.lengths[row] + t - starts[row]
    block = s.tables[row, (pos // b).clamp_max(s.tables.shape[1] - 1).long()]
    slots = torch.where(granted[row] & ~behind, block * b + pos % b, torch.full_like(pos, -1))
    rows = torch.where(behind, torch.full_like(pos, -1), row.to(torch.int32))
    s.free_count_out.copy_(s.free_count - torch.where(granted, need, torch.zeros_like(need)).sum())
    return {"tables": s.tables, "starts": starts, "ends": torch.where(granted, end, s.lengths), "rows": rows, "positions": torch.where(behind, torch.zeros_like(pos), pos),
            "slots": slots, "free_count": s.free_count_out}


def _scale_for(amax):
    """The smallest power of two s, 2^-118 at least, with amax <= 448 s."""
    m, e = torch.frexp(amax)                                  # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(amax > 0, e, torch.full_like(e, LEAST)).clamp_min(LEAST)
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _append(s):
    b = s.block
    block, off = (s.slots // b).long(), s.slots % b
    x = torch.stack([s.k, s.v]).float()                                                    # [2, T, H, D]
    two, tokens, heads, dim = x.shape
    amax = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)           # [2, T, H]
    seen = torch.full((2, s.scale.shape[1], heads), -1.0, device=DEV)
    seen.scatter_reduce_(1, block[None, :, None].expand(2, tokens, heads), amax, "amax")
    fresh = torch.zeros(s.scale.shape[1], dtype=torch.int32, device=DEV).scatter_reduce_(0, block, (off == 0).to(torch.int32), "amax") > 0
    old = s.scale.clone()
    new = torch.maximum(torch.where(fresh[None, :, None], torch.zeros_like(old), old), _scale_for(seen.clamp_min(0)))
    new = torch.where(seen >= 0, new, old)
    # the first block of a row may hold earlier tokens: their codes go to the new scale
    first = s.starts[:-1].long().clamp_max(tokens - 1)
    fb, fo = block[first], off[first]
    before = torch.arange(b, device=DEV)[None] < torch.where(s.new_lens > 0, fo, torch.zeros_like(fo))[:, None]     # [rows, b]
    part = s.kv[:, fb]                                                                     # [2, rows, H, b, D]
    moved = (part.float() * (old[:, fb] / new[:, fb])[..., None, None]).to(F8)
    s.kv.view(torch.uint8)[:, fb] = torch.where(before[None, :, None, :, None], moved.view(torch.uint8), part.view(torch.uint8))
    codes = torch.where(torch.isfinite(x), x / new[:, block][..., None], torch.full_like(x, math.nan)).to(F8)
    s.kv.view(torch.uint8)[:, block, :, off.long()] = codes.view(torch.uint8).transpose(0, 1)
    s.scale.copy_(new)
    return {"kv": s.kv, "scale": s.scale}


def _attend(s):
    rows, b = s.ends.numel(), s.block
    tokens, hq, dim = s.q.shape
    hk = s.kv.shape[2]
    most, longest = s.max_new, max(h + n for h, n in zip(s.held, s.new))
    pages = _need(longest, b)
    table = s.tables[:, :pages].clamp_min(0).long()
    k, v = (s.kv[i, table].float() * s.scale[i, table][..., None, None] for i in (0, 1))    # [rows, pages, hk, b, dim]
    k, v = (x.permute(0, 2, 1, 3, 4).reshape(rows, hk, pages * b, dim) for x in (k, v))
    at = s.starts[:-1, None] + torch.arange(most, device=DEV)[None]
    real = at < s.starts[1:, None]
    at = at.clamp_max(tokens - 1).long()
    q = s.q[at].float().reshape(rows, most, hk, hq // hk, dim).permute(0, 2, 3, 1, 4).reshape(rows, hk, (hq // hk) * most, dim)
    pos = (s.ends - s.new_lens)[:, None] + torch.arange(most, device=DEV)[None]            # position of each new token
    key = torch.arange(pages * b, device=DEV)
    hidden = (key[None, None] > pos[..., None]) | (key[None, None] >= s.ends[:, None, None])
    sc = (q @ k.transpose(-1, -2)).reshape(rows, hk, hq // hk, most, pages * b).mul_(1.0 / math.sqrt(dim))
    sc.masked_fill_(hidden[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    sc.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = sc.sum(-1, keepdim=True)
    v = torch.where((key[None] < s.ends[:, None])[:, None, :, None], v, torch.zeros_like(v))
    o = (sc.reshape(rows, hk, -1, pages * b) @ v).reshape(rows, hk, hq // hk, most, dim) / total.clamp_min(1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(rows, most, hq, dim)
    keep = real[..., None, None]
    to = torch.where(real, at, torch.full_like(at, tokens))
    wide = torch.empty(tokens + 1, hq, dim, dtype=torch.bfloat16, device=DEV)
    wide[to.reshape(-1)] = torch.where(keep, o, torch.zeros_like(o)).reshape(-1, hq, dim).to(torch.bfloat16)
    s.out.copy_(wide[:tokens])
    return s.out


def _select(s):
    r, beams, vocab = s.logits.shape
    x = s.logits.double()                                    # neighbours in the order may be near: 64 bits
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x).clamp_max(3.4028234663852886e38)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    value = s.scores.double()[..., None] + (x - top - (x - top).exp().sum(-1, keepdim=True).log())
    value = torch.where(x == -math.inf, x, value)
    if s.finished is not None:
        only = torch.full_like(value, -math.inf)
        only[..., s.eos] = s.scores.double()
        value = torch.where(s.finished[..., None], only, value)
    best, at = torch.sort(value.reshape(r, beams * vocab), dim=-1, descending=True, stable=True)
    best, at = best[:, :beams], at[:, :beams]
    parent, token = at // vocab, at % vocab
    done = torch.gather(s.finished, 1, parent) | (token == s.eos) if s.finished is not None else torch.zeros_like(parent, dtype=torch.bool)
    return best.float(), parent.to(torch.int32), token.to(torch.int32), done


def _reorder(s):
    rows, width = s.tables.shape
    b = s.block
    j = torch.arange(rows, device=DEV)
    p = (j // s.beams) * s.beams + s.parents.reshape(-1).long()
    length = s.lengths[p]
    full, fill = length // b, length % b
    moved = (p != j) & (fill > 0)
    col = torch.arange(width, device=DEV)[None]
    taken = torch.where(col < ((length + b - 1) // b)[:, None], s.tables[p], torch.full_like(s.tables, -1))
    s.tables_out.copy_(torch.where(moved[:, None] & (col == full[:, None]), s.spare[:, None], taken))
    mine = torch.gather(s.tables, 1, (s.lengths // b).long().clamp_max(width - 1)[:, None])[:, 0]
    left = torch.where(s.lengths % b > 0, mine, torch.full_like(mine, -1))
    s.spare_out.copy_(torch.where(moved, left, s.spare))
    s.lengths_out.copy_(length)
    source = torch.gather(s.tables[p], 1, full.long().clamp_max(width - 1)[:, None])[:, 0].long()
    source = torch.where(moved, source, s.spare.long())      # a row that stays copies its spare block onto itself
    to = s.spare.long()
    raw = s.kv.view(torch.uint8)
    old = raw[:, :, to]
    keep = moved[:, None] & (torch.arange(b, device=DEV)[None] < fill[:, None])
    raw[:, :, to] = torch.where(keep[None, None, :, None, :, None], raw[:, :, source], old)
    s.scale[:, :, to] = s.scale[:, :, source]
    return {"kv": s.kv, "scale": s.scale, "tables": s.tables_out, "lengths": s.lengths_out, "spare": s.spare_out}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """Row by row from the definitions, in 64 bits."""
    s = prepare(case, seed)
    return {"plan": _exact_plan, "append": _exact_append, "attend": _exact_attend, "select": _exact_select, "reorder": _exact_reorder}[s.op](s)


def _exact_plan(s):
    b, tables, free = s.block, s.tables.tolist(), s.free.tolist()
    count = s.free.numel()
    starts, ends, rows, positions, slots = [0], [], [], [], []
    for i, (h, n) in enumerate(zip(s.held, s.new)):
        starts.append(starts[-1] + n)
        for blk in range(_need(h, b), _need(h + n, b)):
            count -= 1
            tables[i][blk] = free[count]
        ends.append(h + n)
        for p in range(h, h + n):
            rows.append(i)
            positions.append(p)
            slots.append(tables[i][p // b] * b + p % b)
    return {"tables": _ints(tables), "starts": _ints(starts), "ends": _ints(ends), "rows": _ints(rows), "positions": _ints(positions), "slots": _ints(slots), "free_count": _ints([count])}


def _exact_append(s):
    b, kv, scale = s.block, s.kv.double(), s.scale.double()
    powers = torch.tensor([2.0 ** e for e in range(LEAST, 122)], dtype=torch.float64, device=DEV)
    at = 0
    for i, (h, n) in enumerate(zip(s.held, s.new)):
        for blk in range(h // b, _need(h + n, b)):
            lo, hi = max(h, blk * b), min(h + n, (blk + 1) * b)
            if lo >= hi:
                continue
            page = int(s.tables[i, blk])
            x = torch.stack([s.k[at + lo - h: at + hi - h], s.v[at + lo - h: at + hi - h]]).double()        # [2, t, H, D]
            want = powers[torch.searchsorted(TOP * powers, x.abs().amax((1, 3)))]                          # [2, H]: the first that suffices
            now = want if lo == blk * b else torch.maximum(want, scale[:, page])
            kv[:, page, :, : lo - blk * b] *= (scale[:, page] / now)[..., None, None]
            kv[:, page, :, lo - blk * b: hi - blk * b] = (x / now[:, None, :, None]).transpose(1, 2)
            scale[:, page] = now
        at += n
    return {"kv": kv, "scale": scale}


def _exact_attend(s):
    b, dim = s.block, s.q.shape[2]
    group = s.q.shape[1] // s.kv.shape[2]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEV)
    at = 0
    for i, (h, n) in enumerate(zip(s.held, s.new)):
        pages = s.tables[i, : _need(h + n, b)].long()
        k, v = ((s.kv[j, pages].double() * s.scale[j, pages].double()[..., None, None]).transpose(0, 1).reshape(s.kv.shape[2], -1, dim)[:, : h + n] for j in (0, 1))
        late = torch.arange(h + n, device=DEV)[None] > (h + torch.arange(n, device=DEV))[:, None]
        for head in range(s.q.shape[1]):
            sc = s.q[at: at + n, head].double() @ k[head // group].T / math.sqrt(dim)
            out[at: at + n, head] = torch.softmax(sc.masked_fill(late, -math.inf), -1) @ v[head // group]
        at += n
    return out


def _exact_select(s):
    r, beams, vocab = s.logits.shape
    best, parents, tokens, done = [], [], [], []
    for i in range(r):
        value = s.scores[i].double()[:, None] + torch.log_softmax(s.logits[i].double(), -1)
        if s.finished is not None:
            for j in range(beams):
                if bool(s.finished[i, j]):
                    value[j] = -math.inf
                    value[j, s.eos] = s.scores[i, j].double()
        v, at = value.reshape(-1).cpu().sort(descending=True, stable=True)
        v, at = v[:beams], at[:beams]
        best.append(v)
        parents.append(at // vocab)
        tokens.append(at % vocab)
        done.append(torch.tensor([s.finished is not None and (bool(s.finished[i, int(a) // vocab]) or int(a) % vocab == s.eos) for a in at]))
    return torch.stack(best), torch.stack(parents), torch.stack(tokens), torch.stack(done)


def _exact_reorder(s):
    b, kv, scale, tables, spare = s.block, s.kv.float(), s.scale.double(), s.tables.tolist(), s.spare.tolist()
    old, left = [list(t) for t in tables], list(spare)
    parents, lengths = s.parents.reshape(-1).tolist(), []
    for j in range(len(spare)):
        p = j // s.beams * s.beams + parents[j]
        n = s.held[p]
        lengths.append(n)
        tables[j] = old[p][: _need(n, b)] + [-1] * (s.width - _need(n, b))
        if p != j and n % b:
            kv[:, :, spare[j], :, : n % b] = kv[:, :, old[p][n // b], :, : n % b]
            scale[:, :, spare[j]] = scale[:, :, old[p][n // b]]
            tables[j][n // b] = spare[j]
            left[j] = old[j][s.held[j] // b]
    return {"kv": kv.double(), "scale": scale, "tables": _ints(tables), "lengths": _ints(lengths), "spare": _ints(left)}
