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
