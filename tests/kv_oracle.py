"""Definitions of the paged 8-bit cache, of attention over it and of beam search, in 64 bits and row by row."""
import math

import numpy as np
import torch

TOP = 448.0


def e4m3(x):
    """Nearest e4m3 value of each element (ties to the even code), |x| <= 448; NaN stays NaN."""
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.maximum(np.where(x == 0, -6, np.floor(np.log2(np.abs(np.where(x == 0, 1, x))))), -6)
    step = np.exp2(e - 3)
    return np.rint(x / step) * step


def scale_for(amax):
    e = -118
    while TOP * 2.0 ** e < amax:
        e += 1
    return 2.0 ** e


def plan(tables, lengths, new, free, count, block, tokens):
    """→ dict of arrays, refused rows; tables is a copy."""
    tables = np.array(tables)
    rows, width = tables.shape
    count = max(0, min(count, len(free)))
    starts, ends = [0], list(lengths)
    row_of, pos, slots = np.full(tokens, -1), np.zeros(tokens, int), np.full(tokens, -1)
    off, taken, refused = 0, 0, []
    for i in range(rows):
        a = starts[-1]
        starts.append(a + max(0, new[i]))
        fits = lengths[i] >= 0 and new[i] >= 0 and lengths[i] + new[i] <= width * block and starts[-1] <= tokens
        have = -(-lengths[i] // block)
        need = -(-(lengths[i] + new[i]) // block) - have if fits else 0
        ok = fits and (need == 0 or off + need <= count)
        if ok:
            for k in range(need):
                tables[i, have + k] = free[count - 1 - off - k]
            taken = off + need if need else taken
            ends[i] = lengths[i] + new[i]
        else:
            refused.append(i)
        off += need
        for t in range(a, min(starts[-1], tokens)):
            row_of[t], pos[t] = i, lengths[i] + t - a
            if ok:
                slots[t] = tables[i, pos[t] // block] * block + pos[t] % block
    return dict(tables=tables, starts=np.array(starts), ends=np.array(ends), rows=row_of, positions=pos, slots=slots, left=count - taken), refused


def append(codes, scale, k, v, slots):
    """codes [2, N, H, bs, D] as values, scale [2, N, H]; returns new copies.  Rounds like the definition."""
    codes, scale = np.array(codes, dtype=np.float64), np.array(scale, dtype=np.float64)
    N, H, bs = codes.shape[1:4]
    x = np.stack([k, v]).astype(np.float64)
    t = 0
    while t < len(slots):
        s = int(slots[t])
        if s < 0 or s >= N * bs:
            t += 1
            continue
        page, off = divmod(s, bs)
        n = 1
        while off + n < bs and t + n < len(slots) and slots[t + n] == s + n:
            n += 1
        for w in range(2):
            for h in range(H):
                run = x[w, t: t + n, h]
                fin = np.isfinite(run)
                now = scale_for(np.abs(run[fin]).max() if fin.any() else 0.0)
                if off:
                    old = scale[w, page, h]
                    now = max(now, old)
                    if now != old:
                        codes[w, page, h, :off] = e4m3(codes[w, page, h, :off] * (old / now))
                codes[w, page, h, off: off + n] = e4m3(np.where(fin, run, np.nan) / now)
                scale[w, page, h] = now
        t += n
    return codes, scale


def attention(q, codes, scale, tables, starts, ends, c, skip=()):
    """→ (o, A): output and, for tolerances, the same sum over magnitudes; rows of tokens without a row stay NaN."""
    q = np.asarray(q, dtype=np.float64)
    T, hq, D = q.shape
    _, N, hk, bs, _ = codes.shape
    o, A = np.full((T, hq, D), np.nan), np.zeros((T, hq, D))
    for i in range(len(ends)):
        a, b, end = int(starts[i]), min(int(starts[i + 1]), T), int(ends[i])
        if i in skip:
            continue
        ids = tables[i][: -(-end // bs)].astype(int)
        kv = [(codes[w, ids] * scale[w, ids][..., None, None]).transpose(1, 0, 2, 3).reshape(hk, -1, D)[:, :end] for w in range(2)]
        for t in range(a, b):
            last = min(end, end - (int(starts[i + 1]) - t) + 1)
            for h in range(hq):
                if last <= 0:
                    o[t, h] = 0
                    continue
                k, v = (x[h // (hq // hk), :last] for x in kv)
                s = k @ q[t, h] * c
                p = np.exp(s - s.max()) if np.isfinite(s).all() else np.full_like(s, np.nan)
                p = p / p.sum()
                o[t, h], A[t, h] = p @ v, p @ np.abs(v)
    return o, A


def select(logits, scores, finished=None, eos=None):
    x = logits.double().cpu()
    R, B, V = x.shape
    x = torch.where(torch.isnan(x), torch.tensor(-math.inf, dtype=torch.float64), x).clamp_max(3.4028234663852886e38)
    out = []
    for r in range(R):
        vals = torch.full((B, V), -math.inf, dtype=torch.float64)
        for b in range(B):
            s = float(scores[r, b])
            if math.isnan(s) or s == -math.inf:
                continue
            if finished is not None and bool(finished[r, b]):
                vals[b, eos] = s
            elif (x[r, b] > -math.inf).any():
                m = x[r, b].max()
                vals[b] = s + (x[r, b] - m - torch.log(torch.exp(x[r, b] - m).sum()))
        v, at = vals.reshape(-1).sort(descending=True, stable=True)
        out.append([(float(v[k]), int(at[k]) // V, int(at[k]) % V) for k in range(B)])
    return out


def reorder(codes, scale, tables, lengths, parents, spare):
    """codes [L, 2, N, H, bs, D]; returns new copies of everything."""
    codes, scale, tables = np.array(codes), np.array(scale), np.array(tables)
    old, oc, os_ = tables.copy(), codes.copy(), scale.copy()
    beams, bs = parents.shape[1], codes.shape[4]
    lens, left = [], list(spare)
    for j, p in enumerate(parents.reshape(-1)):
        src = j // beams * beams + int(p)
        n = int(lengths[src])
        lens.append(n)
        tables[j] = -1
        tables[j, : -(-n // bs)] = old[src, : -(-n // bs)]
        if src != j and n % bs:
            codes[:, :, spare[j], :, : n % bs] = oc[:, :, old[src, n // bs], :, : n % bs]
            scale[:, :, spare[j]] = os_[:, :, old[src, n // bs]]
            tables[j, n // bs] = spare[j]
            left[j] = old[j, lengths[j] // bs] if lengths[j] % bs else -1
    return codes, scale, tables, np.array(lens), np.array(left)
