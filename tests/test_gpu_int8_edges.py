"""8-bit rows on the GPU: the calls at the edge of what the documents allow."""
import pytest
import torch

from circuit_rag import Int8Rows, dequantize_rows

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


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [1, 8, 33, 384, 1000, 5000])
def test_read_of_a_store_without_rows(d, dtype):
    store = Int8Rows(0, d, DEV)
    ids = store.search(_rows(3, d), 4)[1]
    assert (ids == -1).all()
    assert torch.equal(store.read(ids, dtype=dtype), torch.zeros(3, 4, d, dtype=dtype, device=DEV))
    for n in (5, 2000):  # few rows and many
        ids = torch.randint(-3, 4, (n,), device=DEV)
        got = store.read(ids, dtype=dtype)
        assert (got[ids < 0] == 0).all() and got[ids >= 0].isnan().all()
    assert store.read(ids[:0]).shape == (0, d)
    assert dequantize_rows(store.codes, store.scales).shape == (0, d)
