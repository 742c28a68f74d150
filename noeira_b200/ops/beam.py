"""Beam search: selection over beams and vocabulary (csrc/beam.cu), and the cache's states following the beams
(csrc/kv_cache.cu); CPU tensors take the same definitions in PyTorch."""
from __future__ import annotations

import math

import torch

from .._native import check, cuda_lib, raw_stream
from .kvcache import F8, _ints, _need, _on
from .status import status_ptr

MAX_BEAMS = 32
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
    _need(logits.dim() == 3 and logits.numel() > 0, f"logits: [requests, beams, vocab], got {tuple(logits.shape)}")
    requests, beams, vocab = logits.shape
    dev = logits.device
    _need(beams <= MAX_BEAMS and requests * beams < 1 << 31, f"beam_select: at most {MAX_BEAMS} beams, got {beams}")
    _need(scores.dtype is torch.float32 and scores.shape == (requests, beams) and scores.is_contiguous() and scores.device == dev,
          f"scores: contiguous float32 {(requests, beams)}, got {scores.dtype} {tuple(scores.shape)}")
    _need(eos is None or 0 <= eos < vocab, f"eos: a token of {vocab}, got {eos}")
    if finished is not None:
        _need(eos is not None, "finished: needs eos")
        _need(finished.dtype is torch.bool and finished.shape == scores.shape and finished.is_contiguous() and finished.device == dev,
              f"finished: contiguous bool {(requests, beams)}, got {finished.dtype} {tuple(finished.shape)}")
    if not logits.is_cuda:
        return _select_cpu(logits, scores, finished, eos)
    fp32 = logits.dtype is torch.float32
    _need(fp32 or logits.dtype is torch.bfloat16, f"logits: bf16 or fp32, got {logits.dtype}")
    s0, pitch, s2 = logits.stride()
    if beams == 1:
        pitch = s0 if requests > 1 else vocab
    _need((s2 == 1 or vocab == 1) and pitch >= vocab and (requests == 1 or s0 == beams * pitch), f"logits: rows of unit stride at one pitch, got strides {logits.stride()}")
    guard = _on(logits)
    if guard is not None:
        with guard:
            return beam_select(logits, scores, finished, eos)
    out = torch.empty(3, requests, beams, dtype=torch.int32, device=dev)
    done = torch.empty(requests, beams, dtype=torch.bool, device=dev)
    new_scores, parents, tokens = out[0].view(torch.float32), out[1], out[2]
    check(cuda_lib().nb_beam_select(logits.data_ptr(), scores.data_ptr(), None if finished is None else finished.data_ptr(), new_scores.data_ptr(), parents.data_ptr(),
                                    tokens.data_ptr(), done.data_ptr(), requests, beams, vocab, -1 if eos is None else eos, int(fp32), pitch, raw_stream()), "beam_select")
    return new_scores, parents, tokens, done


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
    _need(kv.dtype is F8 and kv.dim() == 6 and kv.shape[1] == 2 and kv.is_contiguous(), f"kv: contiguous {F8} [layers, 2, blocks, heads, block, head_dim], got {kv.dtype} {tuple(kv.shape)}")
    layers, _, blocks, heads, block, dim = kv.shape
    dev = kv.device
    _need(scale.dtype is torch.float32 and scale.shape == kv.shape[:4] and scale.is_contiguous() and scale.device == dev, f"scale: contiguous float32 {tuple(kv.shape[:4])}, got {scale.dtype} {tuple(scale.shape)}")
    _need(dim % 16 == 0 and block > 0, f"head_dim {dim}: a multiple of 16")
    _need(parents.dim() == 2 and tables.dim() == 2 and parents.numel() == tables.shape[0] and parents.numel() > 0, f"parents [requests, beams] over tables [requests * beams, width], got {tuple(parents.shape)} and {tuple(tables.shape)}")
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
    _need(tables_out.data_ptr() != tables.data_ptr() and lengths_out.data_ptr() != lengths.data_ptr() and spare_out.data_ptr() != spare.data_ptr(), "beam_reorder: outputs may not be the inputs")
    if not kv.is_cuda:
        return _reorder_cpu(kv, scale, tables, lengths, parents, spare, tables_out, lengths_out, spare_out)
    guard = _on(kv)
    if guard is not None:
        with guard:
            return beam_reorder(kv, scale, tables, lengths, parents, spare, tables_out, lengths_out, spare_out)
    check(cuda_lib().nb_kv_reorder(
        kv.data_ptr(), scale.data_ptr(), tables.data_ptr(), lengths.data_ptr(), parents.data_ptr(), spare.data_ptr(), tables_out.data_ptr(), lengths_out.data_ptr(),
        spare_out.data_ptr(), 2 * layers, blocks, heads, block, dim, rows, parents.shape[1], width, status_ptr(kv.get_device()), raw_stream()), "kv_reorder")
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
