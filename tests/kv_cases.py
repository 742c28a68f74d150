"""Inputs that the CPU and GPU tests of the paged cache share."""
import numpy as np
import torch

F8 = torch.float8_e4m3fn


def random_codes(shape, seed, nan=False):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=g) * 70).clamp(-448, 448).to(F8)
    if nan:
        x.view(torch.uint8)[torch.rand(shape, generator=g) < 0.1] = 0x7F
    return x


def values(codes):
    return codes.cpu().float().double().numpy()


def paged(lengths, block, seed, spare_blocks=3, extra_width=1):
    """Shuffled tables for rows of the given lengths → (tables int32, number of blocks, unused ids)."""
    need = [-(-n // block) for n in lengths]
    blocks = sum(need) + spare_blocks
    ids = np.random.RandomState(seed).permutation(blocks)
    t = np.full((len(lengths), max(need) + extra_width), -1, dtype=np.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = ids[at: at + n]
        at += n
    return t, blocks, ids[at:]


# held, new tokens per row, query heads, cache heads, head_dim, block
ATTENTION = [
    ([0], [1], 1, 1, 64, 16),                                         # one token that sees itself only
    ([15, 16, 17], [1, 1, 1], 6, 6, 64, 16),                          # around a block's border
    ([639], [1], 6, 6, 64, 16),
    ([5, 0, 300, 63, 64, 65, 1], [1, 1, 1, 1, 1, 1, 1], 15, 5, 64, 32),
    ([1000, 3, 250], [1, 1, 1], 16, 1, 128, 64),                      # sixteen query heads to one
    ([700, 129], [1, 1], 32, 1, 64, 128),                             # more than sixteen
    ([40, 0, 7], [3, 0, 5], 6, 2, 64, 16),                            # a few tokens, a row without new ones
    ([0, 0, 0], [17, 33, 1], 8, 2, 128, 32),                          # short prompts into an empty cache
    ([33], [130], 3, 3, 64, 16),                                      # a chunk over earlier tokens
    ([0, 5], [300, 129], 4, 1, 128, 128),
    ([2000, 77], [1, 257], 4, 2, 64, 64),                             # a single token beside a prompt
    ([0, 1, 511], [128, 127, 256], 12, 12, 128, 16),
    ([3000, 1, 4100], [1, 1, 2], 8, 8, 128, 16),
]

# enough query rows for the tensor cores' kernel: tiles of 256 query rows, several of them, ends inside tiles and key blocks
PROMPTS = [
    ([0], [513], 8, 8, 64, 16),                                       # exactly one token past two tiles
    ([0, 40, 0], [256, 255, 900], 12, 12, 64, 16),
    ([500, 1000], [300, 1], 32, 4, 128, 64),                          # eight heads to one, a single token beside it
    ([0, 127, 128, 3000], [700, 65, 1, 64], 16, 8, 128, 32),
    ([129, 0, 7, 900], [900, 0, 16, 33], 24, 8, 64, 128),
]


def attention_inputs(case, seed=0):
    held, new, hq, hk, dim, block = case
    lengths = [h + n for h, n in zip(held, new)]
    tables, blocks, _ = paged(lengths, block, seed)
    codes = random_codes((2, blocks, hk, block, dim), seed, nan=True)
    # NaN only where no token lies: places behind each row's last, and unused blocks
    live = torch.zeros(blocks, block, dtype=torch.bool)
    for i, n in enumerate(lengths):
        for p in range(n):
            live[tables[i, p // block], p % block] = True
    clean = random_codes((2, blocks, hk, block, dim), seed + 1)
    codes = torch.where(live[None, :, None, :, None], clean.view(torch.uint8), codes.view(torch.uint8)).view(F8)
    g = torch.Generator().manual_seed(seed + 2)
    scale = torch.exp2(torch.randint(-10, -5, (2, blocks, hk), generator=g).float())
    T = sum(new)
    q = (torch.randn(T + 2, hq + 2, dim, generator=g) * 2).bfloat16()        # two tokens and heads more than used: strided views
    starts = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
    return dict(q=q, codes=codes, scale=scale, tables=torch.from_numpy(tables), starts=starts, ends=torch.tensor(lengths, dtype=torch.int32), T=T, max_new=max(new),
                hq=hq, hk=hk, dim=dim, block=block)


# lengths, new tokens, block, free blocks beyond the need, token dimension beyond the need
PLANS = [
    ([0], [1], 16, 0, 0),
    ([15, 16, 0, 31], [1, 1, 0, 2], 16, 2, 3),
    ([3, 64, 100, 0], [70, 1, 28, 0], 32, 5, 0),
    ([0] * 40, list(range(40)), 64, 1, 7),
    ([i % 37 for i in range(700)], [1] * 700, 16, 0, 0),
    ([i * 7 % 300 for i in range(300)], [(i * 13) % 50 for i in range(300)], 128, 9, 1),
    ([0, 5], [3000, 2100], 16, 0, 0),
]
