"""Int8Rows and CircuitRAG(rows="int8"): the 8-bit row operators as a program runs them together."""
import numpy as np
import pytest
import torch

from circuit_rag import CircuitRAG, Int8Rows, quantize_rows

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _rows(n, d, seed=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn(n, d, generator=g, device=DEV)


def _ranked(store, queries, k):
    """Places by the exact products of the stored values, ties to the lower place (64 bits)."""
    qc, qs = quantize_rows(queries)
    values = store.codes.double()
    acc = qc.double() @ values.T
    score = (acc.float() * qs[:, None] * store.scales[None]).double()  # the kernel's roundings
    score[:, store.scales.isnan()] = -np.inf
    order = torch.sort(score, dim=1, descending=True, stable=True)
    return order.values[:, :k], order.indices[:, :k]


@pytest.mark.parametrize("nq,k,block", [(1, 10, 1 << 25), (3, 256, 1 << 25), (70, 7, 1 << 20), (5, 1, 1 << 17)])
def test_search_blocks_and_ties(nq, k, block):
    store = Int8Rows(0, 72, DEV)
    store._BLOCK = block  # several blocks of rows a search
    x = _rows(20000, 72, 1)
    x[5000:5100] = x[:100]  # equal documents: the lower place first
    assert store.append(x[:15000]) == range(0, 15000)
    assert store.append(x[15000:]) == range(15000, 20000)
    assert len(store) == 20000
    q = torch.cat([x[3:4], _rows(nq, 72, 2)])[:nq]
    scores, ids = store.search(q, k)
    assert scores.shape == ids.shape == (nq, k) and ids.dtype == torch.int32
    want_s, want_i = _ranked(store, q, k)
    assert torch.equal(ids.long(), want_i)
    assert torch.equal(scores.double(), want_s)
    if k >= 2:
        assert ids[0, :2].tolist() == [3, 5003]


def test_places_write_remove_and_read():
    store = Int8Rows(100, 33, DEV)
    assert store.scales.isnan().all() and len(store) == 100
    s, i = store.search(_rows(2, 33), 4)
    assert (i == -1).all() and (s == -np.inf).all()
    x = _rows(6, 33, 3)
    store.write(x, torch.tensor([7, -1, 99, 100, 7, 50], device=DEV))
    held = (~store.scales.isnan()).nonzero().flatten().tolist()
    assert held == [7, 50, 99]
    s, i = store.search(x[4:5], 5)
    assert i[0, 0] == 7 and sorted(i[0, :3].tolist()) == [7, 50, 99] and (i[0, 3:] == -1).all()
    back = store.read(i)
    assert back.shape == (1, 5, 33) and (back[0, 3:] == 0).all()
    assert ((back[0, 0] - x[4]).abs() <= x[4].abs().max() / 254 * (1 + 1e-6)).all()  # half a code
    store.remove(torch.tensor([7], device=DEV))
    assert sorted(store.search(x[4:5], 2)[1][0].tolist()) == [50, 99]
    assert store.read(torch.tensor([7], device=DEV)).isnan().all()
    got = store.scores(x[:2])
    assert got.shape == (2, 100) and got[:, [50, 99]].isfinite().all() and got[:, :50].isnan().all()
    assert store.scores(x[:0]).shape == (0, 100) and store.search(x[:0], 3)[1].shape == (0, 3)
    assert Int8Rows(0, 8, DEV).search(_rows(2, 8), 3)[1].tolist() == [[-1] * 3] * 2


def test_append_grows_and_keeps_rows():
    store, parts = Int8Rows(0, 50, DEV), []
    for n in (1, 2, 0, 300, 7, 5000):
        parts.append(_rows(n, 50, n))
        store.append(parts[-1])
    x = torch.cat(parts)
    codes, scales = quantize_rows(x)
    assert torch.equal(store.codes, codes) and torch.equal(store.scales, scales)


def test_store_refusals():
    for bad in (lambda: Int8Rows(-1, 8), lambda: Int8Rows(1, 0), lambda: Int8Rows(1, 16385), lambda: Int8Rows(1 << 31, 8)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        Int8Rows(1, 8, "cpu")
    store = Int8Rows(4, 8, DEV)
    for bad in (lambda: store.append(_rows(2, 9)), lambda: store.write(_rows(2, 9), torch.zeros(2, device=DEV, dtype=torch.int64)),
                lambda: store.write(_rows(2, 8), torch.zeros(3, device=DEV, dtype=torch.int64)),
                lambda: store.search(_rows(1, 9), 2), lambda: store.search(_rows(1, 8), 0),
                lambda: store.search(_rows(1, 8), 257)):
        with pytest.raises(ValueError):
            bad()
    assert len(store) == 4


def test_rag_with_8_bit_rows():
    rng = np.random.default_rng(0)
    vec = {f"doc {i}": rng.standard_normal(48).astype(np.float32) * (i + 1) for i in range(400)}

    def embed(texts):
        return np.stack([vec[t] if t in vec else rng.standard_normal(48).astype(np.float32) for t in texts])

    rag = CircuitRAG(device=DEV, embed_fn=embed, rows="int8")
    assert rag.search("doc 3") == []
    names = list(vec)
    assert rag.add_documents(names[:250], [{"n": i} for i in range(250)]) == list(range(250))
    assert rag.add_documents(names[250:]) == list(range(250, 400))
    unit = np.stack([vec[t] / np.linalg.norm(vec[t].astype(np.float64)) for t in names])
    for t in ("doc 0", "doc 17", "doc 399"):
        got = rag.search(t, k=5)
        q = vec[t] / np.linalg.norm(vec[t].astype(np.float64))
        assert got[0].text == t and len(got) == 5
        for r in got:
            # codes off by at most a half: |error| <= (|q|_1 max|row| + |row|_1 max|q|) / 254, and the product of both
            row = unit[r.id]
            tol = (np.abs(q).sum() * np.abs(row).max() + np.abs(row).sum() * np.abs(q).max()) / 254 * 1.01
            assert abs(r.score - float(q @ row)) <= tol
    assert rag.search("doc 17", k=1)[0].metadata == {"n": 17}
    # feedback moves the query to its documents
    moved = rag.search("doc 5", k=3, feedback=[42])
    assert {r.id for r in moved[:2]} == {5, 42}
    stored = rag.store.read(torch.tensor([42], device=DEV)).double().cpu().numpy()[0]
    v = unit[5] + stored
    want = unit @ (v / np.linalg.norm(v))
    for r in moved:
        assert abs(r.score - want[r.id]) < 0.05  # 48 values: two roundings of half a code each, |v|_1 |u|_max / 254 x 2
    with pytest.raises(ValueError):
        rag.search("doc 5", feedback=[400])


def test_rag_arguments():
    with pytest.raises(ValueError):
        CircuitRAG(device=DEV, embed_fn=lambda t: None, rows="int4")
    plain = CircuitRAG(device=DEV, embed_fn=lambda t: np.eye(8, dtype=np.float32)[: len(t)])
    with pytest.raises(ValueError):
        plain.search("a", feedback=[0])
