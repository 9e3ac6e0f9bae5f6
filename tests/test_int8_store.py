"""The store of 8-bit rows on the host: what its calls do before and after the kernels, on CPU buffers."""
import math

import pytest
import torch

from circuit_rag import Int8Rows


def _host_store(places, dim=8):
    """A store whose buffers lie on the CPU, every place taken (scale 1 + place)."""
    store = Int8Rows.__new__(Int8Rows)
    store.device, store.dim, store._len = torch.device("cpu"), dim, places
    store._codes, store._scales = store._buffers(places)
    store.scales.copy_(torch.arange(places) + 1.0)
    return store


def _held(store):
    return [i for i, s in enumerate(store.scales.tolist()) if not math.isnan(s)]


@pytest.mark.parametrize("slots,left", [
    ([1], [0, 2, 3, 4]), ([-1], [0, 1, 2, 3, 4]), ([5], [0, 1, 2, 3, 4]), ([-1, 4, -7, 0, 1 << 40, -(1 << 63)], [1, 2, 3]),
    ([], [0, 1, 2, 3, 4]), ([2, 2, 2], [0, 1, 3, 4]), ([[0, -1], [5, 3]], [1, 2, 4])])
def test_remove_leaves_other_places_alone(slots, left):
    """-1 (a search's place without a result) and places past the end change nothing, as in write."""
    for dtype in (torch.int64, torch.int32):
        at = torch.tensor(slots, dtype=torch.int64)
        if dtype == torch.int32 and at.numel() and at.abs().max() > 100:
            continue
        store = _host_store(5)
        store.remove(at.to(dtype))
        assert _held(store) == left and len(store) == 5


def test_remove_from_a_store_without_places():
    store = _host_store(0)
    store.remove(torch.tensor([-1, 0, 3]))
    assert _held(store) == [] and len(store) == 0


def test_remove_with_places_in_reserve():
    """Places past the end stay as an append finds them, although buffers are larger than the store."""
    store = _host_store(5)
    store._len = 3
    store.remove(torch.tensor([3, 4]))
    assert store._scales[3:5].tolist() == [4.0, 5.0]


@pytest.mark.parametrize("slots", [torch.tensor([True, False, True]), torch.tensor([0.5]), [0], 0, None])
def test_remove_refuses_what_is_no_place(slots):
    store = _host_store(3)
    with pytest.raises(ValueError):
        store.remove(slots)
    assert _held(store) == [0, 1, 2]
