"""Beam search: selection over beams and vocabulary (csrc/beam.cu), and the cache's states following the beams
(csrc/kv_cache.cu); CPU tensors take the same definitions in PyTorch."""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from .._native import check, cuda_lib, raw_stream
from .kvcache import F8, _ints, _need, _on
from .status import status_ptr

MAX_BEAMS = 32
MAX_VOCAB = 0x7fff0000
_TOP = 3.4028234663852886e38


def beam_select(logits, scores, finished=None, eos=None):
    """The ``beams`` best continuations of every request.

    ``logits`` bf16 or fp32 ``[requests, beams, vocab]`` (rows may be padded: any beam stride with requests ``beams`` strides
    apart), ``scores`` fp32 ``[requests, beams]``: summed log-probabilities, -inf for a beam that does not exist.  The value of
    token ``v`` after beam ``b`` is ``scores[b] + log_softmax(logits[b])[v]``; a beam that is ``finished`` (bool, needs ``eos``)
    has one continuation, ``eos`` at its own score.  Equal values go to the lowest ``b * vocab + v``.  NaN counts as -inf,
    an infinite logit as the largest finite number.

    Returns ``(scores fp32, parents int32, tokens int32, finished bool)``, each ``[requests, beams]``, best first.
    """
    shape = logits.shape
    if len(shape) != 3 or logits.numel() == 0:
        raise ValueError(f"logits: [requests, beams, vocab], got {tuple(shape)}")
    requests, beams, vocab = shape
    dev = logits.get_device()
    if beams > MAX_BEAMS or requests * beams >= 1 << 31 or vocab > MAX_VOCAB:
        raise ValueError(f"beam_select: at most {MAX_BEAMS} beams and {MAX_VOCAB} tokens, got {tuple(shape)}")
    if scores.dtype is not torch.float32 or scores.shape != shape[:2] or not scores.is_contiguous() or scores.get_device() != dev:
        raise ValueError(f"scores: contiguous float32 {(requests, beams)}, got {scores.dtype} {tuple(scores.shape)}")
    if eos is not None and not 0 <= eos < vocab:
        raise ValueError(f"eos: a token of {vocab}, got {eos}")
    if finished is not None:
        if eos is None:
            raise ValueError("finished: needs eos")
        if finished.dtype is not torch.bool or finished.shape != shape[:2] or not finished.is_contiguous() or finished.get_device() != dev:
            raise ValueError(f"finished: contiguous bool {(requests, beams)}, got {finished.dtype} {tuple(finished.shape)}")
    if dev < 0:
        return _select_cpu(logits, scores, finished, eos)
    fp32 = logits.dtype is torch.float32
    if not fp32 and logits.dtype is not torch.bfloat16:
        raise ValueError(f"logits: bf16 or fp32, got {logits.dtype}")
    s0, pitch, s2 = logits.stride()
    if beams == 1:
        pitch = s0 if requests > 1 else vocab
    if (s2 != 1 and vocab > 1) or pitch < vocab or (requests > 1 and s0 != beams * pitch):
        raise ValueError(f"logits: rows of unit stride at one pitch, got strides {logits.stride()}")
    guard = _on(logits)
    if guard is not None:
        with guard:
            return beam_select(logits, scores, finished, eos)
    like = torch.empty_like
    new_scores, parents, tokens, done = like(scores), like(scores, dtype=torch.int32), like(scores, dtype=torch.int32), like(scores, dtype=torch.bool)
    nbytes = _work_bytes(requests, beams, vocab)
    work = scores.new_empty((nbytes + 3) // 4)               # of this call alone
    check(cuda_lib().nb_beam_select(logits.data_ptr(), scores.data_ptr(), None if finished is None else finished.data_ptr(), new_scores.data_ptr(), parents.data_ptr(),
                                    tokens.data_ptr(), done.data_ptr(), requests, beams, vocab, -1 if eos is None else eos, int(fp32), pitch, work.data_ptr(), nbytes,
                                    raw_stream()), "beam_select")
    return new_scores, parents, tokens, done


@functools.lru_cache(maxsize=256)
def _work_bytes(requests, beams, vocab):
    fn = cuda_lib().nb_beam_select_work
    fn.restype = ctypes.c_longlong
    return int(fn(ctypes.c_int(requests), ctypes.c_int(beams), ctypes.c_int(vocab)))


def _select_cpu(logits, scores, finished, eos):
    requests, beams, vocab = logits.shape
    x = logits.double()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x).clamp_max(_TOP)
    score = torch.where(torch.isnan(scores), torch.full_like(scores, -math.inf), scores).double()
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    value = score[..., None] + (x - top - torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    value = torch.where((x == -math.inf) | (score[..., None] == -math.inf), torch.full_like(value, -math.inf), value)
    if finished is not None:
        only = torch.full_like(value, -math.inf)
        only[..., eos] = score
        value = torch.where(finished[..., None], only, value)
    best, at = torch.sort(value.reshape(requests, -1), dim=-1, descending=True, stable=True)
    best, at = best[:, :beams], at[:, :beams]
    parents, tokens = at // vocab, at % vocab
    done = torch.zeros_like(parents, dtype=torch.bool) if eos is None else tokens == eos
    if finished is not None:
        done = done | torch.gather(finished, 1, parents)
    return best.float(), parents.to(torch.int32), tokens.to(torch.int32), done


def beam_reorder(kv, scale, tables, lengths, parents, spare, tables_out=None, lengths_out=None, spare_out=None):
    """Lets the rows of a cache follow the beams that ``beam_select`` kept.

    ``kv`` / ``scale``: all layers, ``[layers, 2, blocks, heads, block, head_dim]`` and ``[layers, 2, blocks, heads]``; ``parents``
    int32 ``[requests, beams]``: row ``r * beams + j`` of the tables continues from row ``r * beams + parents[r, j]``.  Full
    blocks are shared by naming them; a partly filled last block is copied into ``spare[row]`` (int32 ``[rows]``), and the block
    that the row filled so far becomes its next spare (-1 where it had none).  A row that continues itself keeps its blocks.
    The spare blocks have to be distinct and named by no table.  Returns ``(tables, lengths, spare)`` of the next step, written to the ``_out`` tensors if given; these may not be the
    inputs.
    """
    shape, dev = kv.shape, kv.get_device()
    if kv.dtype is not F8 or len(shape) != 6 or shape[1] != 2 or not kv.is_contiguous():
        raise ValueError(f"kv: contiguous {F8} [layers, 2, blocks, heads, block, head_dim], got {kv.dtype} {tuple(shape)}")
    layers, _, blocks, heads, block, dim = shape
    if scale.dtype is not torch.float32 or scale.shape != shape[:4] or not scale.is_contiguous() or scale.get_device() != dev:
        raise ValueError(f"scale: contiguous float32 {tuple(shape[:4])}, got {scale.dtype} {tuple(scale.shape)}")
    if dim % 16 or block <= 0:
        raise ValueError(f"head_dim {dim}: a multiple of 16")
    if parents.dim() != 2 or tables.dim() != 2 or parents.shape[0] * parents.shape[1] != tables.shape[0] or tables.shape[0] == 0:
        raise ValueError(f"parents [requests, beams] over tables [requests * beams, width], got {tuple(parents.shape)} and {tuple(tables.shape)}")
    rows, width = tables.shape
    _ints("tables", tables, dev)
    _ints("lengths", lengths, dev, rows)
    _ints("parents", parents, dev)
    _ints("spare", spare, dev, rows)
    tables_out = torch.empty_like(tables) if tables_out is None else tables_out
    lengths_out = torch.empty_like(lengths) if lengths_out is None else lengths_out
    spare_out = torch.empty_like(spare) if spare_out is None else spare_out
    _ints("tables_out", tables_out, dev, rows * width)
    _ints("lengths_out", lengths_out, dev, rows)
    _ints("spare_out", spare_out, dev, rows)
    tp, lp, sp, tpo, lpo, spo = tables.data_ptr(), lengths.data_ptr(), spare.data_ptr(), tables_out.data_ptr(), lengths_out.data_ptr(), spare_out.data_ptr()
    if tp == tpo or lp == lpo or sp == spo:
        raise ValueError("beam_reorder: outputs may not be the inputs")
    if dev < 0:
        return _reorder_cpu(kv, scale, tables, lengths, parents, spare, tables_out, lengths_out, spare_out)
    guard = _on(kv)
    if guard is not None:
        with guard:
            return beam_reorder(kv, scale, tables, lengths, parents, spare, tables_out, lengths_out, spare_out)
    check(cuda_lib().nb_kv_reorder(kv.data_ptr(), scale.data_ptr(), tp, lp, parents.data_ptr(), sp, tpo, lpo, spo, 2 * layers, blocks, heads, block, dim, rows,
                                   parents.shape[1], width, status_ptr(dev), raw_stream()), "kv_reorder")
    return tables_out, lengths_out, spare_out


def _reorder_cpu(kv, scale, tables, lengths, parents, spare, tables_out, lengths_out, spare_out):
    beams, block, width = parents.shape[1], kv.shape[4], tables.shape[1]
    raw = kv.view(torch.uint8)
    for j, p in enumerate(parents.reshape(-1).tolist()):
        _need(0 <= p < beams, f"parents: row {j} continues from beam {p} of {beams}")
        src = j // beams * beams + p
        n = int(lengths[src])
        full, fill = divmod(n, block)
        tables_out[j] = torch.where(torch.arange(width) < -(-n // block), tables[src], torch.full_like(tables[src], -1))
        lengths_out[j], spare_out[j] = n, spare[j]
        if src != j and fill:
            a, b = int(tables[src, full]), int(spare[j])
            _need(0 <= a < kv.shape[2] and 0 <= b < kv.shape[2], f"beam_reorder: row {j} has no block to copy or no spare block")
            raw[:, :, b, :, :fill] = raw[:, :, a, :, :fill]
            scale[:, :, b] = scale[:, :, a]
            tables_out[j, full] = b
            mine = int(lengths[j])
            spare_out[j] = tables[j, mine // block] if mine % block else -1
    return tables_out, lengths_out, spare_out
