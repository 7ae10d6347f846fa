"""Packed and single-token operators at their edges, as far as that can be seen without a GPU."""
import ctypes

import pytest
import torch

from ossm_b200 import _lib, packed


def test_indices_past_32_bits_stay_out_of_range():
    at = torch.tensor([0, 7, -3, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 40 + 5, -(2 ** 32)])
    got = packed._index("slots", at, at.device)
    assert got.dtype == torch.int32 and got.tolist() == [0, 7, -1] + [2 ** 31 - 1] * 4 + [-1]
    narrow = at[:3].int()
    assert packed._index("slots", narrow, at.device) is narrow
    assert packed._index("slots", torch.arange(8).int()[::2], at.device).tolist() == [0, 2, 4, 6]


def test_library_refuses_a_cache_without_an_entry_for_each_sequence():
    lib = _lib.load()
    p = ctypes.c_void_p(256)
    calls = [lambda count, entries: lib.ossm_b200_selective_scan_packed_forward(
                 p, 8, p, 8, p, p, 4, p, 4, None, 0, None, None, 0, p, None, None, 0, p, p, entries, p, 8, 1, None, None, 0, 4, count,
                 8, 4, 0, 0, None),
             lambda count, entries: lib.ossm_b200_conv1d_silu_packed_forward(
                 p, 8, p, None, p, None, None, 0, p, p, entries, p, 8, 1, 4, count, 8, 4, 0, 0, None),
             lambda count, entries: lib.ossm_b200_selective_scan_step(
                 p, 8, p, 8, p, p, 4, p, 4, None, 0, None, None, 0, None, p, entries, p, 8, count, 8, 4, 0, 0, None),
             lambda count, entries: lib.ossm_b200_conv1d_silu_step(
                 p, 8, p, None, None, p, entries, p, 8, count, 8, 4, 0, 0, None)]
    for call in calls:
        assert call(3, 2) < 0 and "fewer entries than sequences" in lib.ossm_b200_last_error().decode()


@pytest.mark.parametrize("slots, fits", [(None, False), (torch.tensor([1, -1, 0]), True)])
def test_cache_with_fewer_entries_than_sequences(slots, fits):
    cache = torch.zeros(2, 3, 8)
    check = lambda: packed._check_cache("cache", cache, (3, 8), torch.float32, cache.device, 3, slots)
    if fits:
        check()
    else:
        with pytest.raises(RuntimeError, match="2 entries for 3 sequences"):
            check()
    packed._check_cache("cache", cache[:, :0].contiguous(), (0, 8), torch.float32, cache.device, 3, None)   # one tap: no window to lose


@pytest.mark.parametrize("device", ["cpu", "meta"])
def test_cache_is_made_where_the_mixer_lies(device):
    from types import SimpleNamespace

    from ossm_b200.mixer import MambaCache

    weight = torch.empty(32, 8, device=device, dtype=torch.bfloat16)
    cache = MambaCache(SimpleNamespace(in_proj=SimpleNamespace(weight=weight), d_conv=4, d_inner=16, d_state=5), 3)
    assert cache.conv.shape == (3, 3, 16) and cache.conv.dtype == torch.bfloat16 and cache.conv.device.type == device
    assert cache.ssm.shape == (3, 16, 5) and cache.ssm.dtype == torch.float32 and cache.ssm.device.type == device
