"""A small GPT, its logits over the cache, and the same over a whole sequence with keys and values rounded as the cache rounds them."""
import numpy as np
import torch

import kv_oracle as O
from noeira_b200.models.gpt import GPT


def model(device, tie=False, layers=2):
    m = GPT(vocab=64, seq=64, dim=128, layers=layers, heads=2, tie=tie, seed=5)
    g = torch.Generator().manual_seed(2)
    for _, p in m.named_params():                    # weights large enough that attention is not an average
        if p.data.dim() == 2:
            p.data.copy_(torch.randn(p.data.shape, generator=g) * (0.15 if p.data.shape[0] != 64 else 1.0))
            p.version += 1
    return m.to(device).eval()


def sequences():
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 64, (n,), generator=g).tolist() for n in (1, 16, 37, 5)]
    steps = [torch.randint(0, 64, (18,), generator=g).tolist() for _ in prompts]
    return prompts, steps


def cached_logits(m, prompts, steps):
    """[row][n]: logits after the prompt and n of its steps."""
    dev = m.wte.weight.data.device
    rows, out = len(prompts), []
    cache = m.new_cache(rows, 64)
    new = [len(p) for p in prompts]
    ids = [t for p in prompts for t in p]
    for n in range(len(steps[0]) + 1):
        plan = cache.plan(torch.tensor(new, dtype=torch.int32, device=dev), len(ids))
        out.append(m.forward_cached(torch.tensor(ids, device=dev), cache, plan, max_new=max(new)).float().cpu())
        if n < len(steps[0]):
            new, ids = [1] * rows, [s[n] for s in steps]
    return [[o[r] for o in out] for r in range(rows)]


def rounded(x, block):
    """[S, H, D] → what the cache holds of it, in fp64."""
    S, H, D = x.shape
    pages = -(-S // block)
    codes, scale = O.append(np.zeros((2, pages, H, block, D)), np.zeros((2, pages, H)), x, x, list(range(S)))
    return (codes[0] * scale[0][..., None, None]).transpose(0, 2, 1, 3).reshape(-1, H, D)[:S]


@torch.no_grad()
def quantised_logits(m, ids, block):
    """Logits [S, vocab] of one sequence; keys and values rounded, attention in fp64, the rest through the model's own layers."""
    dev = m.wte.weight.data.device
    S = len(ids)
    x = m.wte.forward(torch.tensor(ids, device=dev)) + m.wpe.forward(torch.arange(S, device=dev))
    for b in m.blocks:
        a = b.attn
        qkv = a.qkv.forward(b.n1.forward(x)).reshape(S, 3 * a.h, a.hd)
        q = qkv[:, : a.h].double().cpu()
        k, v = (torch.from_numpy(rounded(t.float().cpu().numpy(), block)) for t in (qkv[:, a.h: 2 * a.h], qkv[:, 2 * a.h:]))
        s = torch.einsum("qhd,khd->hqk", q, k) / a.hd ** 0.5
        s = s.masked_fill(torch.ones(S, S).triu(1).bool(), float("-inf"))
        o = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v).reshape(S, -1).to(device=dev, dtype=qkv.dtype)
        x = a.out.forward(o, residual=x)
        x = b.ffn.forward(b.n2.forward(x), residual=x)
    h = m.ln_f.forward(x)
    if not m.tie:
        return m.head.forward(h).float().cpu()
    W = m.wte.weight
    return (h.float() @ (W.shadow if h.is_cuda else W.data)[: m.vocab, : m.dim].float().t()).cpu()


@torch.no_grad()
def attention_block(device, heads=4, kv_heads=2, head_dim=128):
    """Cached attention of a block with grouped heads, prompts and single tokens of two rows, and the definition in 64 bits."""
    from noeira_b200 import nn
    from noeira_b200.ops.kvcache import PagedKVCache
    nn.manual_seed(3)
    a = nn.SelfAttention(256, heads, kv_heads, head_dim, mask="causal").to(device).eval()
    cache = PagedKVCache(1, kv_heads, head_dim, 20, 2, 60, 16, device=device)
    g = torch.Generator().manual_seed(9)
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    x = [torch.randn(n, 256, generator=g).to(device=device, dtype=dtype) for n in (40, 23)]
    got, at = [[], []], [0, 0]
    for new in ([30, 0], [1, 17], *[[1, 1]] * 6, [3, 0]):
        tokens = torch.cat([x[r][at[r]: at[r] + n] for r, n in enumerate(new)])
        plan = cache.plan(torch.tensor(new, dtype=torch.int32, device=device), len(tokens))
        o = a.forward_cached(tokens, cache, 0, plan, max_new=max(new))
        for r, n in enumerate(new):
            got[r].append(o[sum(new[:r]): sum(new[:r]) + n])
            at[r] += n
    want = []
    for r in range(2):
        S = at[r]
        qkv = a.qkv.forward(x[r][:S]).reshape(S, heads + 2 * kv_heads, head_dim)
        k, v = (torch.from_numpy(rounded(t.float().cpu().numpy(), 16)).repeat_interleave(heads // kv_heads, 1) for t in (qkv[:, heads: heads + kv_heads], qkv[:, heads + kv_heads:]))
        s = torch.einsum("qhd,khd->hqk", qkv[:, :heads].double().cpu(), k) / head_dim ** 0.5
        o = torch.einsum("hqk,khd->qhd", torch.softmax(s.masked_fill(torch.ones(S, S).triu(1).bool(), float("-inf")), -1), v).reshape(S, -1)
        want.append(a.out.forward(o.to(device=device, dtype=dtype)).float().cpu())
    return [torch.cat(t).float().cpu() for t in got], want
