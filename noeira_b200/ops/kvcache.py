"""Paged key / value cache in 8 bits: block tables and slot maps, writing tokens, attention over the cache
(csrc/kv_cache.cu, csrc/kv_attention.cu) and the fp32 forms that CPU tensors take.

A layer of the cache is codes ``float8_e4m3fn [2, blocks, heads, block, head_dim]`` (keys, values) with one fp32 scale per block
and head ``[2, blocks, heads]``; a key or value is code × scale, and scales are powers of two.  A row (one sequence) owns the
blocks that its line of ``tables`` int32 ``[rows, width]`` names; token number ``p`` of the row lies at slot
``tables[row, p // block] * block + p % block``.  The new tokens of a call are ragged: row ``i`` owns tokens
``starts[i] .. starts[i + 1]`` of the token dimension.

None of the calls synchronises.  What only the device can see (no free block, a bad block id) is reported through the status
word (``ops.check_status``) and never touches memory outside the tensors; on CPU tensors, whose forms compute in fp32, the same
raises ``RuntimeError`` or ``ValueError`` (a plan before it changes anything).
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple

import torch

from .._native import check, cuda_lib, raw_stream
from .status import status_ptr

F8 = torch.float8_e4m3fn
F8_TOP = 448.0
LEAST_EXPONENT = -118
BLOCKS = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
MAX_ROWS = 8192
FEW = 64              # query rows of a row and head, up to which the kernel of few query rows does it in any case


class TokenPlan(NamedTuple):
    starts: torch.Tensor       # int32 [rows + 1] first token of each row
    ends: torch.Tensor         # int32 [rows]     tokens that the row holds after the call
    rows: torch.Tensor         # int32 [tokens]   row of each token, -1 behind the last
    positions: torch.Tensor    # int32 [tokens]   place of each token in its row, 0 where it has no slot
    slots: torch.Tensor        # int32 [tokens]   slot of each token, -1 where there is none
    free_count: torch.Tensor   # int32 [1]        free blocks that are left


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _on(t):
    """Guard for a launch on the tensor's own device (its current stream); None where that device is current already."""
    return None if t.get_device() == torch._C._cuda_getDevice() else torch.cuda.device(t.device)


def _ints(name, t, device, numel=None):
    """``device``: the index that ``get_device`` gives, -1 for the CPU."""
    if t.dtype is not torch.int32 or not t.is_contiguous() or t.get_device() != device or (numel is not None and t.numel() != numel):
        raise ValueError(f"{name}: contiguous int32 on device {device}" + (f" with {numel} elements" if numel is not None else "") + f", got {t.dtype} {tuple(t.shape)} on {t.device}")


# ------------------------------------------------------------------------------------------------ plan
def plan_tokens(tables, lengths, new_lens, free, free_count, block, tokens, free_count_out=None, max_len=None, blocks=None) -> TokenPlan:
    """Gives every row the blocks for ``new_lens[i]`` more tokens and every token its slot.

    ``tables`` int32 ``[rows, width]`` is completed in place; ``lengths`` / ``new_lens`` int32 ``[rows]``; ``free`` int32 is a
    stack of free block ids of which the first ``free_count`` (int32 ``[1]``) are there; ``tokens`` is the size of the token
    dimension.  Blocks come off the top of the stack in row order.  A row is refused (slots -1, length unchanged, status word)
    when the stack has too few blocks left for it, when it outgrows its table, ``max_len`` tokens (default: what its table has
    room for) or the token dimension, or when a length is negative; behind a row that the stack could not serve, only rows that
    need no new block are served.  A token whose block's id, in the table or on the stack, is none of the cache's ``blocks``
    (default: as many as have slots) gets slot -1 (status word).  ``free_count`` is updated in place unless ``free_count_out`` is
    given.
    """
    dev = tables.get_device()
    shape = tables.shape
    if len(shape) != 2 or not 0 < shape[0] <= MAX_ROWS or shape[1] == 0:
        raise ValueError(f"tables: int32 [rows <= {MAX_ROWS}, width], got {tuple(shape)}")
    rows, width = shape
    _ints("tables", tables, dev)
    _ints("lengths", lengths, dev, rows)
    _ints("new_lens", new_lens, dev, rows)
    _ints("free", free, dev)
    _ints("free_count", free_count, dev, 1)
    if free_count_out is not None:
        _ints("free_count_out", free_count_out, dev, 1)
    if block not in BLOCKS or not 0 <= tokens <= 0x7fffff00 or width * block > 0x7fffff00:
        raise ValueError(f"block {block}, tokens {tokens}, width {width}: blocks of {BLOCKS} tokens, fewer than 2^31 tokens")
    limit = width * block if max_len is None else min(int(max_len), width * block)
    if limit < 0:
        raise ValueError(f"max_len: not negative, got {max_len}")
    if blocks is None:
        blocks = (1 << 31) // block
    elif not 0 < blocks <= (1 << 31) // block:
        raise ValueError(f"blocks: 1 to 2^31 / {block}, got {blocks}")
    if dev < 0:
        return _plan_cpu(tables, lengths, new_lens, free, free_count, block, tokens, free_count_out, limit, blocks)
    guard = _on(tables)
    if guard is not None:
        with guard:
            return plan_tokens(tables, lengths, new_lens, free, free_count, block, tokens, free_count_out, max_len, blocks)
    if free_count_out is None:
        free_count_out = free_count
    # one allocation; its last word is the kernel's own
    buf = torch.empty(3 * tokens + 2 * rows + 2, dtype=torch.int32, device=tables.device)
    slots, positions, row_of, starts, ends, _ = torch.unsafe_split_with_sizes(buf, (tokens, tokens, tokens, rows + 1, rows, 1))   # integers: no autograd to track views for
    at = buf.data_ptr()
    to = at + 12 * tokens
    check(cuda_lib().nb_kv_plan(
        lengths.data_ptr(), new_lens.data_ptr(), tables.data_ptr(), free.data_ptr(), free_count.data_ptr(), free_count_out.data_ptr(), to, to + 4 * rows + 4,
        at + 8 * tokens, at + 4 * tokens, at, to + 8 * rows + 4, rows, width, block, free.numel(), tokens, blocks, limit, status_ptr(dev), raw_stream()), "kv_plan")
    return TokenPlan(starts, ends, row_of, positions, slots, free_count_out)


def _plan_cpu(tables, lengths, new_lens, free, free_count, block, tokens, free_count_out, limit, blocks):
    given, tables = tables, tables.clone()                   # a call that raises changes nothing
    rows = tables.shape[0]
    count = max(0, min(int(free_count), free.numel()))
    starts, ends = torch.zeros(rows + 1, dtype=torch.int32), lengths.clone()
    row_of, positions, slots = (torch.full((tokens,), v, dtype=torch.int32) for v in (-1, 0, -1))
    at, off, taken, refused, bad = 0, 0, 0, [], []
    for i in range(rows):
        held, new = int(lengths[i]), int(new_lens[i])
        first, at = at, at + max(new, 0)
        starts[i + 1] = min(at, 0x7fffffff)
        fits = held >= 0 and new >= 0 and held + new <= limit and at <= tokens
        need = -(-(held + new) // block) + -held // block if fits else 0
        ok = fits and (need == 0 or off + need <= count)
        if ok:
            have = -(-held // block)
            for k in range(need):
                new_id = int(free[count - 1 - off - k])
                tables[i, have + k] = new_id if 0 <= new_id < blocks else -1
            taken = max(taken, off + need) if need else taken
            ends[i] = held + new
        else:
            refused.append(i)
        off += need
        for t in range(first, min(at, tokens)):
            p = held + t - first
            row_of[t] = i
            if not ok:
                continue
            b = int(tables[i, p // block])
            if 0 <= b < blocks:
                slots[t], positions[t] = b * block + p % block, p
            else:
                bad.append(i)
    if refused:
        raise RuntimeError(f"key / value cache: rows {refused} found no room")
    _need(not bad, f"tables, free: rows {sorted(set(bad))} were given blocks outside the cache")
    out = free_count if free_count_out is None else free_count_out
    out.fill_(count - taken)
    given.copy_(tables)
    return TokenPlan(starts, ends, row_of, positions, slots, out)


# ------------------------------------------------------------------------------------------------ append
def _check_layer(kv, scale):
    """→ (device index, blocks, heads, block, head_dim)"""
    shape, dev = kv.shape, kv.get_device()
    if kv.dtype is not F8 or len(shape) != 5 or shape[0] != 2 or not kv.is_contiguous():
        raise ValueError(f"kv: contiguous {F8} [2, blocks, heads, block, head_dim], got {kv.dtype} {tuple(shape)}")
    if scale.dtype is not torch.float32 or scale.shape != shape[:3] or not scale.is_contiguous() or scale.get_device() != dev:
        raise ValueError(f"scale: contiguous float32 {tuple(shape[:3])} beside kv, got {scale.dtype} {tuple(scale.shape)}")
    _, blocks, heads, block, dim = shape
    if block not in BLOCKS or dim not in HEAD_DIMS:
        raise ValueError(f"block {block} and head_dim {dim}: blocks of {BLOCKS} tokens, heads of {HEAD_DIMS}")
    if blocks * block >= 1 << 31:
        raise ValueError("kv: a cache layer has at most 2^31 - 1 slots")
    return dev, blocks, heads, block, dim


def scale_for(amax: torch.Tensor) -> torch.Tensor:
    """The scale of a block whose largest magnitude is ``amax``: the smallest power of two s >= 2^-118 with amax <= 448 s."""
    m, e = torch.frexp(amax.float())                       # amax = m 2^e with m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(amax > 0, e, torch.full_like(e, LEAST_EXPONENT)).clamp_min(LEAST_EXPONENT)
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def append(kv, scale, k, v, slots) -> None:
    """Writes the keys and values of new tokens into a cache layer.

    ``k`` / ``v`` bf16 ``[tokens, heads, head_dim]`` (any token and head strides, e.g. views of a packed projection), ``slots``
    int32 ``[tokens]``; tokens with a slot outside the cache (-1) are skipped.  The tokens of one block have to be neighbours,
    but for skipped ones, with ascending slots, which may leave places out; no slot may appear twice.  A block's scale is that
    of its largest finite magnitude; a call that writes a block's first token starts the block afresh, one that continues it may
    raise the scale and then moves the codes of the earlier tokens.  Non-finite inputs become NaN and do not count for the
    scale.
    """
    dev, blocks, heads, block, dim = _check_layer(kv, scale)
    shape = k.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim or v.shape != shape:
        raise ValueError(f"k, v: [tokens, {heads}, {dim}], got {tuple(shape)} and {tuple(v.shape)}")
    if k.get_device() != dev or v.get_device() != dev:
        raise ValueError("k, v: on the cache's device")
    _ints("slots", slots, dev, shape[0])
    if dev < 0:
        return _append_cpu(kv, scale, k, v, slots)
    ks, vs = k.stride(), v.stride()
    if k.dtype is not torch.bfloat16 or v.dtype is not torch.bfloat16 or ks[2] != 1 or vs[2] != 1:
        raise ValueError("k, v: bf16 with unit stride over head_dim")
    guard = _on(kv)
    if guard is not None:
        with guard:
            return append(kv, scale, k, v, slots)
    check(cuda_lib().nb_kv_append(k.data_ptr(), v.data_ptr(), kv.data_ptr(), scale.data_ptr(), slots.data_ptr(), shape[0], heads, dim, block, blocks,
                                  ks[0], ks[1], vs[0], vs[1], kv.stride(0), raw_stream()), "kv_append")
    return None


def _encode(x, s):
    return torch.where(torch.isfinite(x), x / s, torch.full_like(x, math.nan)).to(F8)


def _append_cpu(kv, scale, k, v, slots):
    block, limit = kv.shape[3], kv.shape[1] * kv.shape[3]
    x = torch.stack([k, v]).float()
    slot = slots.tolist()
    t = 0
    while t < len(slot):
        if slot[t] < 0 or slot[t] >= limit:
            t += 1
            continue
        page, off = divmod(slot[t], block)
        n = 1
        while off + n < block and t + n < len(slot) and slot[t + n] == slot[t] + n:
            n += 1
        run = x[:, t: t + n]
        now = scale_for(torch.where(torch.isfinite(run), run.abs(), torch.zeros_like(run)).amax((1, 3)))
        if off > 0:
            old = scale[:, page].clone()
            now = torch.maximum(now, old)
            kv[:, page, :, :off] = (kv[:, page, :, :off].float() * (old / now)[..., None, None]).to(F8)
        kv[:, page, :, off: off + n] = _encode(run, now[:, None, :, None]).transpose(1, 2)
        scale[:, page] = now
        t += n


# ------------------------------------------------------------------------------------------------ attention
def paged_attention(q, kv, scale, tables, starts, ends, max_new=None, softmax_scale=None, out=None):
    """Causal attention of new tokens over the cache, which holds them already (``append`` comes first).

    ``q`` bf16 ``[tokens, q_heads, head_dim]`` (any token and head strides); ``q_heads`` a multiple of the cache's heads;
    ``starts`` / ``ends`` as in ``TokenPlan``; the token ``t`` of row ``i`` sees the keys at places ``0 .. ends[i] -
    (starts[i + 1] - t)`` of its row.  ``max_new``: an upper bound of the tokens of one row (default: all); 1 in a decode step.
    Tokens behind ``starts[rows]`` are left as they are in ``out``, which may be ``q``; a token that sees nothing gets zeros.  Scores, maxima and sums
    are fp32; the softmax's weights are rounded to f16 (2^-11) before they multiply the values, and for rows with more than 64
    query rows per head whose values' scales differ by more than 2^20 to bf16 (2^-8).
    """
    dev, blocks, hk, block, dim = _check_layer(kv, scale)
    shape = q.shape
    if len(shape) != 3 or shape[2] != dim or shape[1] == 0 or shape[1] % hk or q.get_device() != dev:
        raise ValueError(f"q: [tokens, a multiple of {hk}, {dim}] on the cache's device, got {tuple(shape)} on {q.device}")
    tokens, hq, _ = shape
    if tables.dim() != 2 or not 0 < tables.shape[0] <= MAX_ROWS or tables.shape[1] == 0:
        raise ValueError(f"tables: int32 [rows <= {MAX_ROWS}, width], got {tuple(tables.shape)}")
    rows, width = tables.shape
    _ints("tables", tables, dev)
    _ints("starts", starts, dev, rows + 1)
    _ints("ends", ends, dev, rows)
    softmax_scale = 1.0 / math.sqrt(dim) if softmax_scale is None else float(softmax_scale)
    max_new = tokens if max_new is None else min(int(max_new), tokens)
    if max_new <= 0 < tokens:
        raise ValueError(f"max_new: at least 1, got {max_new}")
    if not softmax_scale > 0:
        raise ValueError(f"softmax_scale: positive, got {softmax_scale}")
    if dev < 0:
        return _attention_cpu(q, kv, scale, tables, starts, ends, softmax_scale, out)
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=q.device)
    elif out.data_ptr() == q.data_ptr() and max_new * (hq // hk) > FEW:
        q = q.clone()                                        # rows with many query rows may be done twice
    qs, os_ = q.stride(), out.stride()
    if q.dtype is not torch.bfloat16 or qs[2] != 1:
        raise ValueError("q: bf16 with unit stride over head_dim")
    if out.dtype is not torch.bfloat16 or out.shape != shape or os_[2] != 1 or out.get_device() != dev:
        raise ValueError("out: bf16 like q with unit stride over head_dim")
    guard = _on(kv)
    if guard is not None:
        with guard:
            return paged_attention(q, kv, scale, tables, starts, ends, max_new, softmax_scale, out)
    # partial results of this call alone: calls on two streams, or in two graphs, share nothing
    floats = _work_floats(dim, rows, tokens, max_new, hq, hk, block, width, _MODE[0])
    work = scale.new_empty(floats) if floats else None
    check(cuda_lib().nb_kv_attention(
        q.data_ptr(), out.data_ptr(), kv.data_ptr(), scale.data_ptr(), tables.data_ptr(), starts.data_ptr(), ends.data_ptr(), rows, tokens, max_new, hq, hk, dim,
        block, blocks, width, qs[0], qs[1], os_[0], os_[1], kv.stride(0), scale.stride(0), softmax_scale, work.data_ptr() if floats else None, floats, status_ptr(dev), raw_stream()), "kv_attention")
    return out


def set_attention_mode(mode: int) -> int:
    """Kernel of rows with more than 64 query rows per head: by problem size (0, default), the one that reads codes straight into the
    fragments of the matrix instructions and spreads a row's keys over the GPU (1), or the one on 256-row tiles of the tensor
    cores (2).  Returns the previous setting."""
    old = int(cuda_lib().nb_kv_attention_mode(ctypes.c_int(mode)))
    _MODE[0] = mode if 0 <= mode <= 2 else old
    return old


_MODE = [0]


@functools.lru_cache(maxsize=1024)
def _work_floats(dim, rows, tokens, max_new, hq, hk, block, width, mode):
    fn = cuda_lib().nb_kv_attention_work
    fn.restype = ctypes.c_longlong
    return int(fn(*map(ctypes.c_int, (dim, rows, tokens, max_new, hq, hk, block, width))))


def _attention_cpu(q, kv, scale, tables, starts, ends, softmax_scale, out):
    tokens, hq, dim = q.shape
    hk, block = kv.shape[2], kv.shape[3]
    out = torch.empty(tokens, hq, dim) if out is None else out
    for i in range(tables.shape[0]):
        a, b, end = int(starts[i]), min(int(starts[i + 1]), tokens), int(ends[i])
        if b <= a:
            continue
        ids = tables[i, : -(-end // block)].long()
        _need(bool(((ids >= 0) & (ids < kv.shape[1])).all()), f"tables: row {i} names a block outside the cache")
        k, v = ((kv[j, ids].float() * scale[j, ids][..., None, None]).transpose(0, 1).reshape(hk, -1, dim)[:, :end].repeat_interleave(hq // hk, 0) for j in (0, 1))
        see = torch.arange(end)[None] <= (end - (int(starts[i + 1]) - torch.arange(a, b)))[:, None]
        s = (q[a:b].float().transpose(0, 1) @ k.transpose(1, 2) * softmax_scale).masked_fill(~see, -math.inf)
        m = s.amax(-1, keepdim=True) if end else torch.zeros(hq, b - a, 1)
        p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
        nan = torch.isnan(v)                                 # a weight of zero does not hide it
        o = p @ v.masked_fill(nan, 0.0) / p.sum(-1, keepdim=True).clamp_min(1e-30)
        o = o.masked_fill(see.float() @ nan.float() > 0, math.nan)
        out[a:b] = o.transpose(0, 1).to(out.dtype)
    return out


# ------------------------------------------------------------------------------------------------ the cache
class PagedKVCache:
    """Storage, block tables and lengths of a model's cache: ``layers`` cache layers over one table.

    ``rows`` sequences of up to ``max_len`` tokens share ``blocks`` blocks.  ``plan`` makes room for new tokens, ``append`` and
    ``attend`` are the calls of one layer, ``reorder`` lets rows follow the beams of a search, ``reset`` empties rows.  For
    ``reorder`` every row owns a spare block (``spares=True``).  The tensors stay the same all along: captured steps may be replayed
    between other calls.
    """

    def __init__(self, layers, kv_heads, head_dim, blocks, rows, max_len, block=16, device="cuda", spares=False):
        _need(layers > 0 and kv_heads > 0 and blocks > 0 and max_len > 0 and 0 < rows <= MAX_ROWS, "PagedKVCache: sizes have to be positive, rows at most %d" % MAX_ROWS)
        _need(block in BLOCKS and head_dim in HEAD_DIMS, f"block {block} and head_dim {head_dim}: blocks of {BLOCKS} tokens, heads of {HEAD_DIMS}")
        _need(blocks * block < 1 << 31, "PagedKVCache: at most 2^31 - 1 slots")
        self.device = torch.device(device)
        self.layers, self.block, self.blocks, self.rows, self.max_len, self.spares = layers, block, blocks, rows, max_len, spares
        self.kv = torch.zeros(layers, 2, blocks, kv_heads, block, head_dim, dtype=torch.uint8, device=self.device).view(F8)
        self.scale = torch.zeros(layers, 2, blocks, kv_heads, device=self.device)
        ints = dict(dtype=torch.int32, device=self.device)
        self.width = -(-max_len // block)
        # tables, lengths and spare blocks lie together, so that a reorder's are put in their place by one copy: a captured step
        # reads the same tensors before and after it
        self._state, self._next = (torch.full((rows * (self.width + 2),), -1, **ints) for _ in range(2))
        self.tables, self.lengths, self.spare = self._views(self._state)
        self.free, self.free_count = torch.empty(blocks, **ints), torch.empty(1, **ints)
        self.reset()

    def _views(self, state):
        tables, lengths, spare = state.split((self.rows * self.width, self.rows, self.rows))
        return tables.view(self.rows, self.width), lengths, spare

    def reset(self, rows=None) -> None:
        """Empties the given rows (default: all) and collects the free blocks: every block that no row and no spare names.
        Synchronises; called between requests, not between tokens."""
        if rows is None:
            self.lengths.zero_()
            self.tables.fill_(-1)
        else:
            self.lengths[rows] = 0
            self.tables[rows] = -1
        used = torch.zeros(self.blocks + 1, dtype=torch.bool, device=self.device)
        used[self.tables.reshape(-1).long()] = True          # -1 marks the extra last element
        used[self.spare.long()] = True
        left = (~used[:-1]).nonzero().flip(0).reshape(-1).to(torch.int32)
        self.free[: left.numel()] = left
        self.free_count.fill_(left.numel())
        if self.spares:
            self.refill_spares()

    def refill_spares(self) -> None:
        """Gives a spare block to every row that has none."""
        lacks = self.spare < 0
        at = self.free_count - lacks.cumsum(0).to(torch.int32)
        got = torch.where(at >= 0, self.free[at.clamp_min(0).long()], torch.full_like(at, -1))
        self.spare.copy_(torch.where(lacks, got, self.spare))
        self.free_count.copy_((self.free_count - lacks.sum().to(torch.int32)).clamp_min(0))

    def plan(self, new_lens, tokens) -> TokenPlan:
        """Room for ``new_lens[i]`` more tokens in row ``i``; the rows' lengths count them from here on."""
        plan = plan_tokens(self.tables, self.lengths, new_lens, self.free, self.free_count, self.block, tokens, max_len=self.max_len, blocks=self.blocks)
        self.lengths.copy_(plan.ends)
        return plan

    def append(self, layer, k, v, plan) -> None:
        append(self.kv[layer], self.scale[layer], k, v, plan.slots)

    def attend(self, layer, q, plan, max_new=None, softmax_scale=None, out=None):
        return paged_attention(q, self.kv[layer], self.scale[layer], self.tables, plan.starts, plan.ends, max_new, softmax_scale, out)

    def reorder(self, parents) -> None:
        """Row ``r * beams + j`` continues from row ``r * beams + parents[r, j]`` (``ops.beam.beam_reorder``)."""
        from .beam import beam_reorder
        _need(self.spares, "PagedKVCache.reorder: the cache was made without spare blocks (spares=True)")
        beam_reorder(self.kv, self.scale, self.tables, self.lengths, parents, self.spare, *self._views(self._next))
        self._state.copy_(self._next)
