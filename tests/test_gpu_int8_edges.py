"""8-bit rows on the GPU: the calls at the edge of what the documents allow."""
import copy
import pickle
import threading
import time

import numpy as np
import pytest
import torch

from circuit_rag import CircuitRAG, Int8Rows, dequantize_rows, int8, int8_scores, quantize_rows, rms_norm_quantize

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


@pytest.mark.parametrize("nq", [1, 3, 20, 200])
@pytest.mark.parametrize("n", [300, 50000])
def test_a_product_without_a_number_comes_first(n, nq):
    """Empty places and queries without a number have no results; any other NaN (here infinity times a row of zeros) shows."""
    store = Int8Rows(0, 32, DEV)
    x = _rows(n, 32, 1)
    x[7] = 0
    x[9] = float("nan")
    store.append(x)
    store.remove(torch.tensor([11], device=DEV))
    qc, qs = quantize_rows(_rows(nq, 32, 2))
    qs[nq // 2] = float("inf")
    scores, ids = store.search_codes(qc, qs, k=2)
    assert ids[nq // 2, 0] == 7 and scores[nq // 2, 0].isnan()
    rest = torch.arange(nq, device=DEV) != nq // 2
    assert scores[rest].isfinite().all()
    qs[nq // 2] = float("nan")
    scores, ids = store.search_codes(qc, qs, k=2)
    assert (ids[nq // 2] == -1).all() and (scores[nq // 2] == -float("inf")).all() and (ids[rest] >= 0).all()
    for k in range(0, n, 9973):  # the kernels' NaN is the one that ranks above every number
        assert (int8_scores(qc, qs, store.codes, store.scales)[nq // 2, k].view(torch.int32) == 0x7FFFFFFF).all()
    int8.check_products()
    int8.check_products(DEV)


def test_places_stay_on_their_device():
    """A device without an index is the current one when the store is made, not when it grows or searches."""
    store = Int8Rows(2, 16, "cuda")
    assert store.device == torch.device("cuda", torch.cuda.current_device()) == store.codes.device
    assert Int8Rows(2, 16).device == store.device


def test_growth_keeps_memory_that_another_stream_reads():
    n, d = 20000, 512
    store = Int8Rows(0, d, DEV)
    x = _rows(n, d, 1)
    store.append(x)
    want = store.scores(x[:3])
    old = store._made[0].data_ptr(), store._made[1].data_ptr()
    size = store._made[0].shape
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000_000)  # about half a second
        got = store.scores(x[:3])
    assert store.append(x[:1]) == range(n, n + 1)  # the buffers are full: new ones
    taken = [torch.full(size, 99, dtype=torch.int8, device=DEV) for _ in range(3)]
    small = [torch.full((n + 1,), 99.0, device=DEV) for _ in range(3)]
    assert not side.query()  # the products are still to come
    assert old[0] not in {t.data_ptr() for t in taken} and old[1] not in {t.data_ptr() for t in small}
    side.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(store.scores(x[:3])[:, :n], want)


def test_a_captured_search_outlives_growth():
    store = Int8Rows(0, 64, DEV)
    x = _rows(5000, 64, 1)
    store.append(x)
    q = x[7:9].clone()
    want = store.search(q, 3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = store.search(q, 3)
        with pytest.raises(RuntimeError):
            store.append(x)
    assert store.append(x) == range(5000, 10000)
    taken = [torch.full((5000, 64), 99, dtype=torch.int8, device=DEV) for _ in range(3)]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    del taken


def test_forward_gradients_are_refused():
    x = _rows(4, 32)
    codes, scales = quantize_rows(x)
    with torch.autograd.forward_ad.dual_level():
        dual = [torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, x[0].clone(), scales)]
        for call in (lambda: quantize_rows(dual[0]), lambda: quantize_rows(dual[0][:, 1:]), lambda: rms_norm_quantize(dual[0]),
                     lambda: rms_norm_quantize(x, residual=dual[0]), lambda: rms_norm_quantize(x, weight=dual[1]),
                     lambda: dequantize_rows(codes, dual[2]), lambda: int8_scores(codes, dual[2], codes, scales),
                     lambda: int8_scores(codes, scales, codes, dual[2]),
                     lambda: int8_scores(codes, scales, codes, scales, bias=dual[2]),
                     lambda: quantize_rows(x, out=(codes, dual[2]))):
            with pytest.raises(RuntimeError):
                call()
            with pytest.raises(RuntimeError), torch.no_grad():  # which leaves forward mode on
                call()
        plain = torch.autograd.forward_ad.unpack_dual(dual[0]).primal
        assert torch.equal(quantize_rows(plain)[0], codes)
    for transform in (lambda f: torch.func.jvp(f, (x,), (x,)), lambda f: torch.func.grad(f)(x), lambda f: torch.func.vmap(f)(x[None])):
        with pytest.raises(RuntimeError):
            transform(lambda t: quantize_rows(t)[1].sum())


def test_results_that_ask_for_a_gradient_are_refused():
    codes, scales = quantize_rows(_rows(4, 32))
    values, products = (torch.empty(4, n, device=DEV).requires_grad_() for n in (32, 4))
    for out in (values, values * 1):  # a leaf, and one with a history that the call would belie
        with pytest.raises(RuntimeError):
            dequantize_rows(codes, scales, out=out)
    for out in (products, products * 1):
        with pytest.raises(RuntimeError):
            int8_scores(codes, scales, codes, scales, out=out)
    with torch.no_grad():
        assert dequantize_rows(codes, scales, out=values) is values
        int8_scores(codes, scales, codes, scales, out=products)


def test_writing_is_known_to_autograd():
    """What a call writes in place cannot be taken for the values that an earlier operation kept for its gradient."""
    x = _rows(4, 32)
    codes, scales = quantize_rows(x)
    store = Int8Rows(0, 32, DEV)
    store.append(x)
    values, products = torch.ones(4, 32, device=DEV), torch.ones(4, 4, device=DEV)
    slots = torch.arange(4, device=DEV)
    for kept, write in ((values, lambda: dequantize_rows(codes, scales, out=values)),
                        (products, lambda: int8_scores(codes, scales, codes, scales, out=products)),
                        (scales, lambda: quantize_rows(2 * x, out=(codes, scales))),
                        (scales, lambda: rms_norm_quantize(x, out=(codes, scales))),
                        (store.scales, lambda: store.write(2 * x, slots))):
        w = torch.ones_like(kept, requires_grad=True)
        loss = (w * kept).sum()
        write()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    before = codes._version, scales._version
    quantize_rows(x[:0], out=(codes[:0], scales[:0]))
    int8_scores(codes, scales, codes, scales)
    dequantize_rows(codes, scales)
    assert (codes._version, scales._version) == before  # nothing was written
    quantize_rows(x, out=(codes, scales))
    assert codes._version > before[0] and scales._version > before[1]
    with torch.inference_mode():
        kept = quantize_rows(x)
        out = torch.empty(4, 32, device=DEV)
        quantize_rows(2 * x, out=kept)
    quantize_rows(2 * x, out=kept)  # tensors without a version
    assert dequantize_rows(*kept, out=out) is out


def test_search_of_many_queries_in_bounded_memory():
    store = Int8Rows(0, 32, DEV)
    store.append(_rows(20000, 32, 1))
    q = _rows(70001, 32, 2)  # more than a call of the products takes
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    scores, ids = store.search(q, 5)
    torch.cuda.synchronize()
    # 2^25 scores of 4 bytes, a few whole numbers of 8 of each, and a sort of these
    assert torch.cuda.max_memory_allocated() - before < 16 * 8 * (1 << 25)
    assert scores.shape == ids.shape == (70001, 5)
    for a in (0, 2040, 2048, 65535, 69990):
        want = store.search(q[a:a + 11], 5)
        assert torch.equal(ids[a:a + 11], want[1]) and torch.equal(scores[a:a + 11], want[0])


def test_tensors_that_stand_for_their_negative():
    """The imaginary part of a conjugate lies in memory with the other sign."""
    z = torch.complex(_rows(300, 40, 1), _rows(300, 40, 2))
    for cut in (slice(0, 40), slice(0, 1)):  # one value a row: any stride is read in place
        rows = z[:, cut].conj().imag
        assert rows.is_neg()
        want = quantize_rows(rows.resolve_neg().contiguous())
        for got in (quantize_rows(rows), quantize_rows(torch._neg_view(-rows.clone()))):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        weight = torch.complex(rows[0].clone(), rows[1].clone()).conj().imag
        got = rms_norm_quantize(rows, residual=rows, weight=weight)
        plain = rows.clone()
        for a, b in zip(got, rms_norm_quantize(plain, residual=plain, weight=weight.clone())):
            assert torch.equal(a, b)
    codes, scales = want
    bias = z[:, 0].conj().imag
    assert torch.equal(int8_scores(codes, scales, codes, scales, bias=bias),
                       int8_scores(codes, scales, codes, scales, bias=bias.clone()))
    assert torch.equal(int8_scores(codes, scales, codes, scales, bias=torch._neg_view(-bias)),
                       int8_scores(codes, scales, codes, scales, bias=bias.clone()))
    for call in (lambda out: dequantize_rows(codes, scales, out=out),
                 lambda out: int8_scores(codes, scales, codes[:1], scales[:1], out=out)):
        with pytest.raises(ValueError):
            call(z[:, :1].conj().imag)
    with pytest.raises(ValueError):
        quantize_rows(plain, out=(codes, torch._neg_view(scales)))


def test_feedback_does_not_depend_on_the_length_of_the_query():
    g = torch.Generator().manual_seed(3)
    vectors = {f"doc {i}": torch.randn(48, generator=g).numpy() for i in range(300)}
    sizes = {"": 1.0, " long": 1e30, " short": 1e-30}

    def embed(texts):
        found = [(vectors[t[:t.index("#")]], sizes[t[t.index("#") + 1:]]) for t in texts]
        return np.stack([v * np.float32(size) for v, size in found])

    rag = CircuitRAG(device=DEV, embed_fn=embed, rows="int8")
    rag.add_documents([f"doc {i}#" for i in range(300)])
    want = rag.search("doc 5#", k=4, feedback=[42, 7])
    assert want[0].id == 5  # random directions: 1 / 1.5^(1/2) against its own document
    for size in (" long", " short"):
        got = rag.search("doc 5#" + size, k=4, feedback=[42, 7])
        assert [r.id for r in got] == [r.id for r in want]
        # the same query but for the rounding of its values: a code may differ by one, the score by less than 1 / 127 for it
        assert all(abs(a.score - b.score) < 0.02 for a, b in zip(got, want))


def test_status_waits_for_its_stream_only():
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(1_000_000_000)  # about half a second on the default stream
    with torch.cuda.stream(side):
        int8.check_products()
    assert not torch.cuda.default_stream().query()
    int8.check_products()
    assert torch.cuda.default_stream().query()


@pytest.mark.parametrize("call", ["quantize", "dequantize", "scores"])
def test_other_threads_run_while_a_launch_waits(call):
    """Behind about a thousand pending launches a further one waits: other Python threads go on meanwhile."""
    x = _rows(4, 32)
    codes, scales = quantize_rows(x)
    out, products = torch.empty(4, 32, device=DEV), torch.empty(4, 4, device=DEV)
    todo = {"quantize": lambda: quantize_rows(x, out=(codes, scales)), "dequantize": lambda: dequantize_rows(codes, scales, out=out),
            "scores": lambda: int8_scores(codes, scales, codes, scales, out=products)}[call]
    todo()
    torch.cuda.synchronize()
    gaps, stop = [0.0], threading.Event()

    def tick():
        last = time.perf_counter()
        while not stop.is_set():
            time.sleep(0.001)
            now = time.perf_counter()
            gaps[0], last = max(gaps[0], now - last), now

    thread = threading.Thread(target=tick)
    thread.start()
    try:
        time.sleep(0.05)
        gaps[0] = 0.0
        longest = 0.0
        torch.cuda._sleep(1_500_000_000)  # about three quarters of a second
        for _ in range(3000):
            start = time.perf_counter()
            todo()
            longest = max(longest, time.perf_counter() - start)
        torch.cuda.synchronize()
    finally:
        stop.set()
        thread.join()
    assert longest < 0.2 or gaps[0] < longest / 2, (longest, gaps[0])


def test_a_thread_searches_while_another_appends():
    store = Int8Rows(0, 64, DEV)
    x = _rows(30000, 64, 1)
    store.append(x[:50])
    torch.cuda.synchronize()
    failed, stop = [], threading.Event()

    def search():
        try:
            q = x[:3].clone()
            while not stop.is_set():
                scores, ids = store.search(q, 3)
                if ids[:, 0].tolist() != [0, 1, 2]:
                    failed.append(ids)
        except Exception as e:  # shown by the main thread
            failed.append(e)

    threads = [threading.Thread(target=search) for _ in range(2)]
    for t in threads:
        t.start()
    for a in range(50, 30000, 599):
        store.append(x[a:a + 599])
    stop.set()
    for t in threads:
        t.join()
    assert not failed, failed[0]
    assert torch.equal(store.scales, quantize_rows(x)[1])


def test_a_copy_of_a_store_is_its_own():
    store = Int8Rows(0, 24, DEV)
    x = _rows(10, 24, 1)
    store.append(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        copies = [copy.deepcopy(store), pickle.loads(pickle.dumps(store))]
        for other in copies:
            assert other._made[2] == side.cuda_stream  # its memory is this stream's
            other.append(x)
    side.synchronize()
    store.remove(torch.tensor([3], device=DEV))
    for other in copies:
        assert len(other) == 20 and len(store) == 10
        assert torch.equal(other.scales, quantize_rows(x)[1].repeat(2))
