"""8-bit rows on the GPU: the calls at the edge of what the documents allow."""
import pytest
import torch

from circuit_rag import Int8Rows

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _rows(n, d, seed=0, dtype=torch.float32):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn(n, d, generator=g, device=DEV).to(dtype)


def _held(store):
    return (~store.scales.isnan()).nonzero().flatten().tolist()


def test_remove_skips_what_is_outside_the_store():
    store = Int8Rows(0, 40, DEV)
    x = _rows(6, 40)
    store.append(x)
    ids = store.search(x[2:3], 9)[1]  # six places and three -1
    assert (ids[0, 6:] == -1).all()
    store.remove(ids[:, 6:])
    store.remove(torch.tensor([6, 7, 1 << 40, -5], device=DEV))
    store.remove(torch.tensor([6]))  # from the host
    assert _held(store) == [0, 1, 2, 3, 4, 5]
    store.remove(ids[:, [0, 8]])
    assert _held(store) == [0, 1, 3, 4, 5]
    assert store.append(x[:1]) == range(6, 7) and _held(store) == [0, 1, 3, 4, 5, 6]
    at = torch.tensor([0, -1], device=DEV)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        store.remove(at)
    at.copy_(torch.tensor([4, 9], device=DEV))
    graph.replay()
    torch.cuda.synchronize()
    assert _held(store) == [0, 1, 3, 5, 6]
