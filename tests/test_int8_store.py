"""The store of 8-bit rows on the host: what its calls do before and after the kernels, on CPU buffers."""
import contextlib
import math

import numpy as np
import pytest
import torch

from circuit_rag import CircuitRAG, Int8Rows, _native, int8


@pytest.fixture(autouse=True)
def _one_stream(monkeypatch):
    monkeypatch.setattr(int8, "_stream", lambda device: 1, raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def _host_store(places, dim=8):
    """A store whose buffers lie on the CPU, every place taken (scale 1 + place)."""
    store = Int8Rows.__new__(Int8Rows)
    store._in_graph, store._captured = False, []
    store.device, store.dim, store._len = torch.device("cpu"), dim, places
    store._made = *store._buffers(places), 1
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
    assert store._made[1][3:5].tolist() == [4.0, 5.0]


@pytest.mark.parametrize("slots", [torch.tensor([True, False, True]), torch.tensor([0.5]), [0], 0, None])
def test_remove_refuses_what_is_no_place(slots):
    store = _host_store(3)
    with pytest.raises(ValueError):
        store.remove(slots)
    assert _held(store) == [0, 1, 2]


def _search(store, products, query_scales, k, monkeypatch):
    """search_codes with given products, as if the kernel had written them."""
    def fake(qc, qs, codes, scales, **kw):
        a = (codes.data_ptr() - store._made[0].data_ptr()) // store._made[0].shape[1]
        return products[:, a:a + codes.shape[0]].clone()

    monkeypatch.setattr(int8, "int8_scores", fake)
    return store.search_codes(torch.zeros(products.shape[0], store.dim, dtype=torch.int8), query_scales, k=k)


def test_a_product_that_gave_up_is_not_an_empty_place(monkeypatch):
    """NaN at a place with a row is a failure that shows; NaN at an empty place, or of a query without a number, is
    no result."""
    nan, inf = float("nan"), float("inf")
    store = _host_store(4)
    store.remove(torch.tensor([1]))
    products = torch.tensor([[3.0, nan, 5.0, nan], [1.0, nan, -inf, 2.0], [nan, nan, nan, nan], [nan, nan, nan, nan]])
    scores, ids = _search(store, products, torch.tensor([1.0, 1.0, nan, 1.0]), 4, monkeypatch)
    assert ids.tolist() == [[3, 2, 0, -1], [3, 0, 2, -1], [-1] * 4, [0, 2, 3, -1]]
    assert scores[0, 0].isnan() and scores[0, 1:].tolist() == [5.0, 3.0, -inf]
    assert scores[1].tolist() == [2.0, 1.0, -inf, -inf]
    assert scores[2].tolist() == [-inf] * 4
    assert scores[3, :3].isnan().all() and scores[3, 3] == -inf


def test_status_reaches_python(monkeypatch):
    class Lib:
        calls = []

        def circuit_op_int8_status(self, stream):
            self.calls.append(stream)
            return -4 if len(self.calls) > 1 else 0

    fake = Lib()
    monkeypatch.setattr(_native, "lib", lambda: fake)
    monkeypatch.setattr(_native, "last_error", lambda: "a bounded wait gave up")
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: type("S", (), {"cuda_stream": 7})())
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    int8.check_products()
    with pytest.raises(_native.NativeLibraryError, match="gave up"):
        int8.check_products()
    assert fake.calls == [7, 7]


def test_rag_reports_a_product_that_gave_up(monkeypatch):
    rag = CircuitRAG(device="cpu", embed_fn=lambda texts: np.ones((len(texts), 8), np.float32), rows="int8")
    rag.texts, rag.metadatas, rag.store = list("abcde"), [{}] * 5, _host_store(5)
    results = [(torch.tensor([2.0, 1.0, -math.inf]), torch.tensor([4, 0, -1], dtype=torch.int32))]
    monkeypatch.setattr(rag, "_search_rows", lambda q, k, feedback: results[-1])
    checked = []
    monkeypatch.setattr("circuit_rag.rag.check_products", lambda device: checked.append(device))
    assert [r.id for r in rag.search("q", k=3)] == [4, 0] and checked == []
    results.append((torch.tensor([math.nan, 1.0, -math.inf]), torch.tensor([3, 0, -1], dtype=torch.int32)))
    with pytest.raises(RuntimeError):
        rag.search("q", k=3)
    assert checked == [rag.store.device]


def test_a_growing_store_stays_on_its_device(monkeypatch):
    """A device without an index means the current one: it is looked up once, when the store is made."""
    asked, current = [], [torch.device("cuda", 3)]
    host = {name: getattr(torch, name) for name in ("zeros", "full", "empty")}

    class Placed:  # a tensor that says where it would lie
        def __init__(self, tensor, device):
            self.tensor, self.device, self.shape = tensor, device, tensor.shape

    def make(name):
        def made(*args, device=None, **kw):
            device = torch.device(device)
            asked.append(device if device.index is not None else current[0])
            return Placed(host[name](*args, **kw), asked[-1])
        return made

    for name in host:
        monkeypatch.setattr(torch, name, make(name))
    store = Int8Rows(2, 8, "cuda")
    current[0] = torch.device("cuda", 0)  # another device is current by now
    codes, scales = store._buffers(9)
    assert store.device == torch.device("cuda", 3) and set(asked) == {store.device}


def _streams(store, monkeypatch, capturing=False):
    """Makes `store` believe in streams 1 (its own), 2, ...: returns the current one's number as a list, and the log of
    (buffer, stream) that the allocator is told of."""
    now, log = [1], []
    stream = type("Stream", (), {"__init__": lambda self, n: setattr(self, "n", n)})
    monkeypatch.setattr(int8, "_stream", lambda device: now[0])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: stream(now[0]))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda self, s: log.append((self.data_ptr(), s.n)))
    monkeypatch.setattr(int8, "quantize_rows", lambda *a, **kw: (torch.zeros(1, 8, dtype=torch.int8), torch.zeros(1)))
    monkeypatch.setattr(int8, "dequantize_rows", lambda *a, **kw: None)
    monkeypatch.setattr(int8, "int8_scores", lambda qc, qs, codes, scales, **kw: torch.zeros(len(qc), len(codes)))
    return now, log


CALLS = {
    "read": lambda s: s.read(torch.zeros(1, dtype=torch.int64)), "scores": lambda s: s.scores(torch.zeros(1, 8)),
    "search": lambda s: s.search(torch.zeros(1, 8), 2), "search_codes": lambda s: s.search_codes(
        torch.zeros(1, 8, dtype=torch.int8), torch.zeros(1), 2),
    "write": lambda s: s.write(torch.zeros(1, 8), torch.zeros(1, dtype=torch.int64)),
    "remove": lambda s: s.remove(torch.zeros(1, dtype=torch.int64)), "append": lambda s: s.append(torch.zeros(9, 8)),
    "codes": lambda s: s.codes, "scales": lambda s: s.scales}


@pytest.mark.parametrize("call", CALLS)
def test_memory_is_kept_for_the_streams_that_use_it(call, monkeypatch):
    """Growth drops the old buffers: the allocator knows every stream that may still read or write them."""
    store = _host_store(4)
    buffers = {store._made[0].data_ptr(), store._made[1].data_ptr()}
    now, log = _streams(store, monkeypatch)
    CALLS[call](store)
    assert log == []  # its own stream: the allocator orders that by itself
    store = _host_store(4)
    buffers = {store._made[0].data_ptr(), store._made[1].data_ptr()}
    now, log = _streams(store, monkeypatch)
    now[0] = 5
    CALLS[call](store)
    assert {b for b, s in log} == buffers and {s for b, s in log} == {5}
    if call == "append":
        assert store._made[2] == 5 and len(store) == 13


def test_buffers_of_a_captured_call_outlive_growth(monkeypatch):
    store = _host_store(4)
    now, log = _streams(store, monkeypatch, capturing=True)
    now[0] = 9
    CALLS["search"](store)
    with pytest.raises(RuntimeError):
        CALLS["append"](store)  # would copy the rows of now at every replay
    assert len(store) == 4
    old = store._made[0]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    CALLS["append"](store)
    assert len(store) == 13 and store._captured[0][0] is old
    CALLS["append"](store)
    CALLS["append"](store)
    assert len(store._captured) == 1  # buffers of no graph are not kept


@pytest.mark.parametrize("places", [0, 4])
def test_search_checks_its_queries(places):
    """Also where nothing is multiplied: a store without places, no queries."""
    store = _host_store(places)
    good = torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2)
    for codes, scales in ((torch.zeros(2, 9, dtype=torch.int8), good[1]), (good[0], torch.zeros(3)), (good[0][0], good[1]),
                          (good[0].float(), good[1]), (good[0], good[1].double()), (good[0], good[1][:, None]),
                          (torch.zeros(0, 9, dtype=torch.int8), torch.zeros(0))):
        with pytest.raises(ValueError):
            store.search_codes(codes, scales, k=2)
    scores, ids = store.search_codes(good[0][:0], good[1][:0], k=2)
    assert scores.shape == ids.shape == (0, 2) and ids.dtype == torch.int32


def test_search_of_many_queries_keeps_its_block(monkeypatch):
    """The scores ranked at a time stay within a block however many queries there are."""
    store, most = _host_store(5000), []
    monkeypatch.setattr(int8, "int8_scores", lambda qc, qs, codes, scales: most.append(len(qc) * len(codes)) or
                        qs[:, None] * scales[None])
    store._BLOCK = 1 << 16
    for nq in (1, 3, 700, 65535 // 16):
        scales = 1.0 + torch.arange(nq) % 7
        scores, ids = store.search_codes(torch.zeros(nq, 8, dtype=torch.int8), scales, k=3)
        assert max(most) <= 1 << 16, nq
        assert ids.tolist() == [[4999, 4998, 4997]] * nq
        assert torch.equal(scores, scales[:, None] * torch.tensor([5000.0, 4999.0, 4998.0]))


def test_rag_without_documents_finds_nothing():
    rag = CircuitRAG(device="cpu", embed_fn=lambda texts: np.ones((len(texts), 8), np.float32), rows="int8")
    rag.store = _host_store(0)  # as adding an empty list leaves it
    assert rag.search("q") == []


def test_zeros_of_both_signs_are_a_tie(monkeypatch):
    """A product that underflows keeps its sign; it is no smaller than a zero."""
    store = _host_store(6)
    tiny = 2.0 ** -149
    products = torch.tensor([[-0.0, 0.0, -0.0, tiny, -tiny, 0.0], [-tiny, -0.0, -2.0, -1.0, -math.inf, math.inf]])
    scores, ids = _search(store, products, torch.ones(2), 6, monkeypatch)
    assert ids.tolist() == [[3, 0, 1, 2, 5, 4], [5, 1, 0, 3, 2, 4]]
    assert scores.tolist() == [[tiny, 0.0, 0.0, 0.0, 0.0, -tiny], [math.inf, 0.0, -tiny, -1.0, -2.0, -math.inf]]
