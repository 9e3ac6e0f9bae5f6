"""What the 8-bit row operators of this package are measured on.

Five operators, each in its plain form (torch, 32 bits) and as the package's own call:

  quantize  rows to 8-bit codes with one scale a row, and the values they stand for
  norm      root-mean-square norm of rows + residual, to 8-bit codes with one scale a row
  write     rows quantised into the slots of a row store and read back from there
  read      rows of a store read back by the ids that a search returned
  scores    queries quantised and multiplied with all rows of a store

A code is rint(127 u / max|u|) of the real quotient, ties to even; a scale is max|u| / 127, for the norm divided by
the root of mean(v^2) + eps.  Negative slots and ids are empty places; of equal slots the last row stays.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
MOST_FLOPS = 6.3e13  # of the largest product
MOST_ROW_BYTES = 800e6  # of the largest store that a product reads


def _ops():
    package = sys.modules.get("circuit_rag")
    if package is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "circuit-rag_b200"))
        import circuit_rag as package
    return package


def listed():
    return [
        # a small corpus taken into 8 bits as a whole (5,183 embeddings of 384)
        {"name": "quantize 5183x384 f32", "op": "quantize", "n": 5183, "d": 384, "t": "f32", "pad": 0},
        # a large batch of half-precision embeddings that lie inside a wider tensor, odd row count
        {"name": "quantize 100001x768 f16 wide", "op": "quantize", "n": 100001, "d": 768, "t": "f16", "pad": 32},
        # one query moved towards its feedback and normalised: the latency of one row
        {"name": "norm 1x384 f32", "op": "norm", "n": 1, "d": 384, "t": "f32", "pad": 0},
        # the last norm of an encoder over the tokens of a batch of passages
        {"name": "norm 65536x1024 bf16", "op": "norm", "n": 65536, "d": 1024, "t": "bf16", "pad": 0},
        # a few new or changed documents, one of them twice, at their slots of a store of 200,000
        {"name": "write 37x1024 bf16", "op": "write", "n": 37, "d": 1024, "t": "bf16", "rows": 200000},
        # a fifth of a store of a million rows renewed
        {"name": "write 200000x384 f32", "op": "write", "n": 200000, "d": 384, "t": "f32", "rows": 1000000},
        # the ten results of one query read back
        {"name": "read 10x384 f32", "op": "read", "n": 10, "d": 384, "t": "f32", "rows": 50000},
        # 100 results for each of 1,024 queries, for a model that reads bf16
        {"name": "read 102400x384 bf16", "op": "read", "n": 102400, "d": 384, "t": "bf16", "rows": 2000000},
        # one query against a small corpus: latency
        {"name": "scores 1x5183x384", "op": "scores", "q": 1, "n": 5183, "d": 384, "t": "f32", "o": "f32", "bias": False},
        # one query against two million rows: the rows' bytes
        {"name": "scores 1x2000000x384", "op": "scores", "q": 1, "n": 2000000, "d": 384, "t": "f32", "o": "f32", "bias": False},
        # a test set of 300 queries against a small corpus, with a prior for each row
        {"name": "scores 300x5183x384 bias", "op": "scores", "q": 300, "n": 5183, "d": 384, "t": "f32", "o": "f32", "bias": True},
        # a serving batch against 40,000 rows of wider embeddings: the product's operations
        {"name": "scores 1024x40000x768 bf16", "op": "scores", "q": 1024, "n": 40000, "d": 768, "t": "bf16", "o": "bf16", "bias": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _dim(rng, lo, hi):
    d = _log(rng, lo, hi)
    return d if rng.random() < 0.4 else max(lo, d // 16 * 16)


def draw(rng):
    op = rng.choice(["quantize", "norm", "write", "read", "scores", "scores"])
    t = rng.choice(["f32", "bf16", "f16"])
    if op in ("quantize", "norm"):
        d = _dim(rng, 16, 8192)
        n = _log(rng, 1, max(1, int(67e6 // d)))
        return {"op": op, "n": n, "d": d, "t": t, "pad": rng.choice([0, 0, 1, 8, 64])}
    d = _dim(rng, 16, 2048)
    if op in ("write", "read"):
        n = _log(rng, 1, max(1, int(76e6 // d)))
        rows = _log(rng, max(1000, n), max(2000, n, int(384e6 // d)))
        return {"op": op, "n": n, "d": d, "t": t, "rows": rows}
    q = _log(rng, 1, 1024)
    most = min(MOST_ROW_BYTES / d, MOST_FLOPS / (2.0 * d * q), 160e6 / q)
    return {"op": op, "q": q, "n": _log(rng, 1000, max(1000, int(most))), "d": d, "t": t,
            "o": rng.choice(["f32", "bf16", "f16"]), "bias": rng.random() < 0.3}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _embeddings(n, d, g):
    """Rows of unit length around a common direction, as embeddings of text lie."""
    x = torch.randn(n, d, generator=g, device="cuda")
    x.add_(torch.randn(1, d, generator=g, device="cuda"))
    return x.div_(x.norm(dim=1, keepdim=True))


def _store(n, d, g):
    """Codes and scales of n embeddings, as a program keeps them: each row padded to a multiple of 16 bytes."""
    codes = torch.zeros(n, -(-d // 16) * 16, dtype=torch.int8, device="cuda")
    scales = torch.empty(n, dtype=torch.float32, device="cuda")
    for a in range(0, n, 1 << 18):
        x = _embeddings(min(n - a, 1 << 18), d, g)
        m = x.abs().amax(1)
        codes[a:a + len(x), :d] = torch.round(x * (127 / m)[:, None]).to(torch.int8)
        scales[a:a + len(x)] = m / 127
    return codes[:, :d], scales


def prepare(case, seed):
    g, d, t = _gen(seed), case["d"], TYPES[case["t"]]
    s = {"case": case}
    if case["op"] == "quantize":
        s["x"] = _wide(_embeddings(case["n"], d, g).to(t), case["pad"])
    elif case["op"] == "norm":
        # hidden states: a few channels much larger than the others
        gain = 1 + 20 * (torch.rand(d, generator=g, device="cuda") < 0.01)
        s["x"] = _wide((torch.randn(case["n"], d, generator=g, device="cuda") * gain).to(t), case["pad"])
        s["r"] = torch.randn(case["n"], d, generator=g, device="cuda").to(t)
        s["w"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(t)
    elif case["op"] == "write":
        s["codes"], s["scales"] = _store(case["rows"], d, g)
        s["x"] = _embeddings(case["n"], d, g).to(t)
        slots = torch.randperm(case["rows"], generator=g, device="cuda")[:case["n"]]
        if case["n"] > 3:  # a document that changed twice, and a place of a padded batch
            slots[-1] = slots[0]
            slots[case["n"] // 2] = -1
        s["slots"] = slots
    elif case["op"] == "read":
        s["codes"], s["scales"] = _store(case["rows"], d, g)
        ids = torch.randint(0, case["rows"], (case["n"],), generator=g, device="cuda", dtype=torch.int32)
        if case["n"] > 3:
            ids[-1] = -1
        s["ids"] = ids
    else:
        s["codes"], s["scales"] = _store(case["n"], d, g)
        s["x"] = _embeddings(case["q"], d, g).to(t)
        s["bias"] = 0.05 * torch.randn(case["n"], generator=g, device="cuda") if case["bias"] else None
    return s


def _wide(x, pad):
    """The same rows inside a tensor with `pad` more columns."""
    if not pad:
        return x
    y = torch.zeros(x.shape[0], x.shape[1] + pad, dtype=x.dtype, device=x.device)
    y[:, :x.shape[1]] = x
    return y[:, :x.shape[1]]


def _codes(u):
    """Codes (as 32-bit numbers) and max|u| of the rows of u.  The quotient is taken in 64 bits: values next to a half."""
    m = u.abs().amax(1, keepdim=True)
    return torch.round(u * 127.0 / torch.where(m > 0, m, 1)).float(), m[:, 0]


def run(s):
    case = s["case"]
    op, t = case["op"], TYPES[case["t"]]
    if own:
        c = _ops()
        if op == "quantize":
            codes, scales = c.quantize_rows(s["x"])
            return {"values": c.dequantize_rows(codes, scales, dtype=t), "scales": scales}
        if op == "norm":
            codes, scales, summed = c.rms_norm_quantize(s["x"], residual=s["r"], weight=s["w"], eps=EPS)
            return {"values": c.dequantize_rows(codes, scales, dtype=t), "scales": scales, "summed": summed}
        if op == "write":
            c.quantize_rows(s["x"], slots=s["slots"], out=(s["codes"], s["scales"]))
            return {"values": c.dequantize_rows(s["codes"], s["scales"], s["slots"], dtype=t), "scales": s["scales"]}
        if op == "read":
            return c.dequantize_rows(s["codes"], s["scales"], s["ids"], dtype=t)
        codes, scales = c.quantize_rows(s["x"])
        return c.int8_scores(codes, scales, s["codes"], s["scales"], bias=s["bias"], dtype=TYPES[case["o"]])
    if op == "quantize":
        codes, m = _codes(s["x"].double())
        scales = m.float() / 127
        return {"values": (codes * scales[:, None]).to(t), "scales": scales}
    if op == "norm":
        summed = (s["x"].float() + s["r"].float()).to(t)
        v = summed.float()
        codes, m = _codes(v.double() * s["w"].double())
        scales = m.float() / 127 / torch.sqrt((v * v).mean(1) + EPS)
        return {"values": (codes * scales[:, None]).to(t), "scales": scales, "summed": summed}
    if op == "write":
        codes, m = _codes(s["x"].double())
        _put(s["codes"], s["scales"], s["slots"], codes, m.float() / 127)
        return {"values": _get(s["codes"], s["scales"], s["slots"], t), "scales": s["scales"]}
    if op == "read":
        return _get(s["codes"], s["scales"], s["ids"], t)
    codes, m = _codes(s["x"].double())
    out = codes @ s["codes"].float().T
    out *= (m.float() / 127)[:, None]
    out *= s["scales"]
    if s["bias"] is not None:
        out += s["bias"]
    return out.to(TYPES[case["o"]])


def _put(codes, scales, slots, new_codes, new_scales):
    """Rows into their slots: none at a negative one, the last of equal ones."""
    i = torch.arange(len(slots), device=slots.device)
    valid = slots >= 0
    at = torch.where(valid, slots, slots.index_select(0, valid.int().argmax().view(1)))  # an empty place repeats a row that is written anyway
    last = torch.full((codes.shape[0],), -1, device=slots.device)
    last.scatter_reduce_(0, at, torch.where(valid, i, -1), "amax")
    row = last[at]
    codes[at] = new_codes[row].to(torch.int8)
    scales[at] = new_scales[row]


def _get(codes, scales, ids, t):
    at = ids.long().clamp(min=0)
    out = codes[at].float() * scales[at][:, None]
    return torch.where((ids >= 0)[:, None], out, 0).to(t)


def exact(case, seed):
    s, t = prepare(case, seed), TYPES[case["t"]]
    op = case["op"]

    def quantised(u):  # codes and the rows' largest magnitude, in 64 bits
        top = torch.linalg.vector_norm(u, ord=math.inf, dim=1)
        return (u * 127 / top.clamp(min=5e-324).unsqueeze(1)).round(), top

    if op == "norm":
        v = (s["x"].double() + s["r"].double()).to(t).double()
        c, top = quantised(v * s["w"].double())
        scale = top / (127 * (v.square().sum(1) / case["d"] + EPS).sqrt())
        return {"values": c * scale.unsqueeze(1), "scales": scale, "summed": v}
    if op == "read":
        known = s["ids"].long() * (s["ids"] >= 0)
        return s["codes"][known].double() * (s["scales"][known].double() * (s["ids"] >= 0)).unsqueeze(1)
    c, top = quantised(s["x"].double())
    scale = top / 127
    if op == "quantize":
        return {"values": c * scale.unsqueeze(1), "scales": scale}
    if op == "write":
        scales = s["scales"].double()
        at = s["slots"].tolist()
        last = {slot: i for i, slot in enumerate(at) if slot >= 0}
        scales[torch.tensor(list(last.keys()), device="cuda")] = scale[torch.tensor(list(last.values()), device="cuda")]
        row = torch.tensor([last.get(slot, -1) for slot in at], device="cuda")
        values = torch.where((row >= 0).unsqueeze(1), (c * scale.unsqueeze(1))[row.clamp(min=0)], 0)
        return {"values": values, "scales": scales}
    left, out = c * scale.unsqueeze(1), torch.empty(case["q"], case["n"], dtype=torch.float64, device="cuda")
    for a in range(0, case["n"], 1 << 18):
        b = slice(a, a + (1 << 18))
        out[:, b] = left @ (s["codes"][b].double() * s["scales"][b].double().unsqueeze(1)).T
    return out if s["bias"] is None else out + s["bias"].double()


def work(case):
    op, d, e = case["op"], case["d"], BYTES[case["t"]]
    if op == "scores":
        q, n = case["q"], case["n"]
        return {"bytes": q * d * e + n * (d + 4) + q * n * BYTES[case["o"]] + (4 * n if case["bias"] else 0), "flops": 2 * q * n * d}
    n = case["n"]
    if op == "read":
        return {"bytes": n * (4 + d + 4 + d * e), "flops": n * d}
    if op == "quantize":  # codes and scales written; the values are what comes back
        return {"bytes": n * (d * e + d + 4 + d * e), "flops": 3 * n * d}
    if op == "norm":  # rows and residual read; sum, codes, scales and values written
        return {"bytes": n * (4 * d * e + d + 4) + d * e, "flops": 7 * n * d}
    return {"bytes": n * (8 + d * e + d + 4 + d * e), "flops": 4 * n * d}
