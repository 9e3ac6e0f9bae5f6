"""Text-in / text-out wrapper (reference circuit_rag/rag.py:11-65), with
incremental document adds instead of a full rebuild per call.

The embedding model is out of scope for the search path and sentence-
transformers is an optional dependency: CircuitRAG imports it only when it is
constructed without an ``embed_fn``.  Any callable mapping a list of strings to
a float32 [n, D] array can be passed instead.
"""
from dataclasses import dataclass, field
from typing import Any, Callable, Dict, List, Optional

import numpy as np
import torch

from circuit_rag.hierarchy.build import build_circuit_index
from circuit_rag.int8 import Int8Rows, check_products, rms_norm_quantize
from circuit_rag.search import circuit_search


@dataclass
class SearchResult:
    id: int
    score: float
    text: str
    metadata: Dict[str, Any] = field(default_factory=dict)


class CircuitRAG:
    def __init__(self, embedding_model: str = "BAAI/bge-small-en-v1.5", device: Optional[str] = None,
                 embed_fn: Optional[Callable[[List[str]], np.ndarray]] = None, rows: str = "float32"):
        if rows not in ("float32", "int8"):
            raise ValueError('rows must be "float32" or "int8"')
        self.rows = rows
        self.store: Optional[Int8Rows] = None
        self.device = device or ("cuda" if torch.cuda.is_available() else "cpu")
        if embed_fn is None:
            from sentence_transformers import SentenceTransformer  # optional dependency

            model = SentenceTransformer(embedding_model, device=self.device)
            embed_fn = lambda texts: model.encode(texts, normalize_embeddings=True, convert_to_numpy=True)
        self._embed = embed_fn
        self.texts: List[str] = []
        self.metadatas: List[Dict[str, Any]] = []
        self._vectors: Optional[np.ndarray] = None
        self.index = None
        self._built_n = 0
        self.appended_rows = 0

    # appended rows beyond this fraction of the last full build trigger a rebuild
    REBUILD_FRACTION = 0.5

    def add_documents(self, texts: List[str], metadatas: Optional[List[Dict[str, Any]]] = None) -> List[int]:
        """Embed and add documents; returns their ids (reference rag.py:33-45).

        The reference rebuilds the whole index on every call.  Here new
        documents are appended to the existing hierarchy (CircuitIndex.append:
        nearest root, new child, certificates recomputed) until the appended
        rows exceed REBUILD_FRACTION of the rows of the last full build; then
        the index is rebuilt with the reference's size rule (rag.py:47-55)."""
        texts = list(texts)
        if metadatas is None:
            metadatas = [{} for _ in range(len(texts))]
        elif len(metadatas) != len(texts):
            raise ValueError("metadatas must be the same length as texts")
        new_vecs = np.asarray(self._embed(texts), dtype=np.float32)
        start_id = len(self.texts)
        if self.rows == "int8":
            if self.store is None:
                self.store = Int8Rows(0, new_vecs.shape[1], self.device)
            # unit length: scores are cosines
            self.store.append(torch.from_numpy(new_vecs).to(self.store.device), normalize=True)
            self.texts.extend(texts)
            self.metadatas.extend(metadatas)
            return list(range(start_id, len(self.texts)))
        self.texts.extend(texts)
        self.metadatas.extend(metadatas)
        if self._vectors is None:
            self._vectors = new_vecs
        else:
            self._vectors = np.concatenate([self._vectors, new_vecs], axis=0)
        n = len(self._vectors)
        if self.index is not None and (n - self._built_n) <= self.REBUILD_FRACTION * self._built_n:
            self.index.append(new_vecs, np.arange(start_id, n, dtype=np.int32))
            self.appended_rows = n - self._built_n
        else:
            self._rebuild()
        return list(range(start_id, n))

    def _rebuild(self):
        n = len(self._vectors)
        roots = int(max(1, min(64, n // 256)))
        children = int(max(1, min(16, n // (roots * 16))))
        self.index = build_circuit_index(self._vectors, num_roots=roots, children_per_root=children,
                                         rank=min(8, self._vectors.shape[1]), device=self.device)
        self._built_n = n
        self.appended_rows = 0

    def search(self, query: str, k: int = 5, feedback: Optional[List[int]] = None) -> List[SearchResult]:
        """The k best documents (reference rag.py:57-65).  feedback (8-bit rows only): ids of documents found
        relevant; the query (at unit length) is moved by their mean before it is compared."""
        if feedback and self.rows != "int8":
            raise ValueError('feedback needs rows="int8"')
        if (self.index is None and self.store is None) or not self.texts:
            return []
        q = torch.from_numpy(np.asarray(self._embed([query]), dtype=np.float32)[0])
        k = min(k, len(self.texts))
        if self.rows == "int8":
            scores, ids = self._search_rows(q.to(self.store.device)[None], k, feedback or [])
        else:
            scores, ids, _ = circuit_search(q, self.index, k=k)
        scores, ids = scores.tolist(), ids.tolist()
        if self.rows == "int8" and any(s != s for s in scores):  # not a missing document: a product was not computed
            check_products(self.store.device)
            raise RuntimeError("a product of the query and a document is not a number")
        return [SearchResult(id=int(i), score=float(s), text=self.texts[int(i)], metadata=self.metadatas[int(i)])
                for s, i in zip(scores, ids) if i >= 0]

    def _search_rows(self, q: torch.Tensor, k: int, feedback: List[int]):
        if any(not 0 <= i < len(self.texts) for i in feedback):
            raise ValueError("feedback must be ids of documents")
        if feedback:
            ids = torch.tensor(feedback, dtype=torch.int64, device=q.device)
            mean = self.store.read(ids).mean(0, keepdim=True)
            wide = q.double()  # squares of 32 bits may leave their range
            q = (wide / wide.norm().clamp(min=torch.finfo(wide.dtype).tiny)).to(q.dtype)  # as long as each document
            # the root-mean-square norm times dim^-1/2: unit length again
            unit = torch.full((self.store.dim,), self.store.dim ** -0.5, device=q.device)
            codes, scales, _ = rms_norm_quantize(q, residual=mean, weight=unit, eps=0.0)
            scores, found = self.store.search_codes(codes, scales, k=k)
        else:
            scores, found = self.store.search(q, k=k, normalize=True)
        return scores[0], found[0]
