"""Packed and single-token operators at their edges, as far as that can be seen without a GPU."""

import torch

from ossm_b200 import packed


def test_indices_past_32_bits_stay_out_of_range():
    at = torch.tensor([0, 7, -3, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 40 + 5, -(2 ** 32)])
    got = packed._index("slots", at, at.device)
    assert got.dtype == torch.int32 and got.tolist() == [0, 7, -1] + [2 ** 31 - 1] * 4 + [-1]
    narrow = at[:3].int()
    assert packed._index("slots", narrow, at.device) is narrow
    assert packed._index("slots", torch.arange(8).int()[::2], at.device).tolist() == [0, 2, 4, 6]
