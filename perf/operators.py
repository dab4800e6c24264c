"""The microscaled 4-bit floating-point operators of pion_b200, as they are measured.

A store holds embedding rows in one of two formats, quantised as the rows are written:

* ``mx``: blocks of 32 elements, each an e2m1 code (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign), one
  power of two per block (e8m0: the exponent of the block's largest magnitude less 2);
* ``nv``: blocks of 16 e2m1 codes, an e4m3 scale s per block and a float32 scale g per row:
  g = amax / 2688, s = e4m3(bmax / float32(6 g)), element = e2m1(x / float32(s g)).

Every rounding is to nearest, ties to even, of the exact quotient.  A row with a NaN or an
infinity leaves its slot empty (g = NaN): it reads as NaN, scores -inf and is never found.

``write`` cases quantise rows into slots of a store and read those slots back; ``scores`` cases
quantise a batch of queries and take their products with every row of a store; ``knn`` cases
also keep the k best rows of each query, by (score, lowest slot), where a score is the exact
sum rounded once to float32.

The store as a program keeps it: codes uint8 [slots, dp / 2], two codes a byte, the lower
nibble first, dp the dimension rounded up to 128; scales uint8 [ceil(slots / 128)][atoms][32]
[4][4]: block b of row r at tile r / 128, atom b / 4, [r % 32][r % 128 / 32][b % 4];
row_scale float32 [slots] (g; 1 in ``mx``); norm_max float32 [1], at least every row's norm;
claim int32 [slots], zero between calls.
"""
import functools
import math

import torch

own = False

BLOCK = {"mx": 32, "nv": 16}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # one document's embedding arrives and goes into its slot: latency
        {"name": "write_one_row", "op": "write", "format": "nv", "slots": 65536, "rows": 1,
         "dim": 1536, "type": "f32", "out": "f32", "pad": 0},
        # a burst of new embeddings from a bf16 encoder, to scattered slots
        {"name": "write_burst_bf16", "op": "write", "format": "mx", "slots": 65536, "rows": 4096,
         "dim": 1536, "type": "bf16", "out": "bf16", "pad": 0},
        # an odd dimension, rows inside a wider buffer (row stride dim + pad)
        {"name": "write_odd_f16", "op": "write", "format": "nv", "slots": 100003, "rows": 50021,
         "dim": 777, "type": "f16", "out": "f16", "pad": 7},
        # a whole index loaded at once
        {"name": "write_index", "op": "write", "format": "nv", "slots": 262144, "rows": 262144,
         "dim": 1536, "type": "f32", "out": "f32", "pad": 0},
        # one query against a small collection: latency
        {"name": "scores_small", "op": "scores", "format": "mx", "n": 1000, "nq": 1, "dim": 1536,
         "type": "f32", "out": "f32"},
        # one query against every row of a million: the memory-bound end
        {"name": "scores_one_query", "op": "scores", "format": "nv", "n": 1000000, "nq": 1,
         "dim": 1536, "type": "f32", "out": "f32"},
        # ragged sizes, half-precision scores for a later stage
        {"name": "scores_ragged_bf16", "op": "scores", "format": "mx", "n": 200003, "nq": 77,
         "dim": 1000, "type": "bf16", "out": "bf16"},
        # the score matrix of a batch: the compute-bound end
        {"name": "scores_batch", "op": "scores", "format": "nv", "n": 262144, "nq": 1024,
         "dim": 1536, "type": "f32", "out": "f32"},
        # the k nearest of a small collection: latency
        {"name": "knn_small", "op": "knn", "format": "nv", "n": 5000, "nq": 1, "dim": 1536,
         "k": 10, "type": "f32"},
        # the k nearest of a million for one query (one FT.SEARCH)
        {"name": "knn_one_query", "op": "knn", "format": "mx", "n": 1000000, "nq": 1, "dim": 1536,
         "k": 10, "type": "f32"},
        # an odd number of rows, a shortlist of 64 for a later rerank
        {"name": "knn_ragged", "op": "knn", "format": "mx", "n": 300007, "nq": 60, "dim": 400,
         "k": 64, "type": "bf16"},
        # the benchmark's batch: 1M rows, 1024 queries, k = 10
        {"name": "knn_batch", "op": "knn", "format": "nv", "n": 1000000, "nq": 1024, "dim": 1536,
         "k": 10, "type": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "scores", "knn"])
    fmt = rng.choice(["mx", "nv"])
    typ = rng.choice(["f32", "bf16", "f16"])
    dim = rng.choice([rng.randint(16, 512), rng.randint(512, 2048), 384, 768, 1536])
    if op == "write":
        rows = min(_log(rng, 1, 262144), 400000000 // dim)
        return {"op": op, "format": fmt, "slots": rows + _log(rng, 1, 65536), "rows": rows,
                "dim": dim, "type": typ, "out": rng.choice(["f32", "bf16", "f16"]),
                "pad": rng.choice([0, 0, 1, 8, 64])}
    n = min(_log(rng, 500, 1000000), 1536000000 // dim)
    if op == "scores":
        nq = min(_log(rng, 1, 1024), max(1, 268435456 // n), max(1, 400000000000 // (n * dim)))
        return {"op": op, "format": fmt, "n": n, "nq": nq, "dim": dim, "type": typ,
                "out": rng.choice(["f32", "bf16", "f16"])}
    return {"op": op, "format": fmt, "n": n, "nq": _log(rng, 1, 1024), "dim": dim,
            "k": rng.choice([1, 10, 10, rng.randint(1, 64), rng.randint(1, 256)]), "type": typ}


# ------------------------------------------------------------- plain forms --
def _pad_dim(dim):
    return (dim + 127) // 128 * 128


def _e4m3(y):
    """The nearest e4m3 number (ties to even) of y in [0, 448 (1 + 2^-20)], in float64."""
    step = torch.exp2(torch.clamp(torch.frexp(y)[1].double() - 1.0, min=-6.0) - 3.0)
    return torch.clamp(torch.round(y / step) * step, max=448.0)


def _quantise(x, fmt):
    """Rows x [n, dim] of any type -> (codes uint8 [n, dp] with the sign in bit 3, block
    scales float32 [n, blocks] and their bytes, g float32 [n])."""
    n, dim = x.shape
    dp, block = _pad_dim(dim), BLOCK[fmt]
    x = x.float()
    fine = torch.isfinite(x).all(1)
    x = torch.where(fine[:, None], x, 0.0)
    x = torch.nn.functional.pad(x, (0, dp - dim)).view(n, dp // block, block)
    bmax = x.abs().amax(2)
    if fmt == "mx":
        e = torch.clamp(torch.frexp(bmax)[1] - 3, -127, 125)
        e = torch.where(bmax > 0, e, -127)
        bits = (e + 127).to(torch.uint8)
        scale = torch.ldexp(torch.ones_like(bmax, dtype=torch.float64), e).float()
        g = torch.ones(n, device=x.device)
        d = scale
    else:
        amax = bmax.amax(1)
        live = amax >= 2.0 ** -100
        # a division by a number would be a product with its rounded reciprocal
        g = torch.where(live, amax / torch.full_like(amax, 2688.0), 0.0)
        h = torch.where(live, 6.0 * g, 1.0)
        s = torch.where(live[:, None], _e4m3(bmax.double() / h.double()[:, None]), 0.0)
        scale = s.float()
        bits = scale.to(torch.float8_e4m3fn).view(torch.uint8)
        d = scale * g[:, None]
    y, d = x.abs().double(), d.double()[:, :, None]
    code = (y > 0.25 * d).to(torch.uint8)
    code += y >= 0.75 * d
    code += y > 1.25 * d
    code += y >= 1.75 * d
    code += y > 2.5 * d
    code += y >= 3.5 * d
    code += y > 5.0 * d
    code = torch.where((d > 0) & (x != 0), code + 8 * (x < 0).to(torch.uint8), 0)
    g = torch.where(fine, g, float("nan"))
    bits = torch.where(fine[:, None], bits, 0)
    return code.view(n, dp), scale, bits, g


def _scale_at(slots, atoms):
    """Where the scale bytes of rows `slots` lie: int64 [n, 4 * atoms]."""
    b = torch.arange(4 * atoms, device=slots.device)
    r = slots[:, None]
    return ((((r // 128) * atoms + b // 4) * 32 + r % 32) * 4 + r % 128 // 32) * 4 + b % 4


def _put(st, slots, code, bits, g):
    st["codes"][slots] = code[:, 0::2] | (code[:, 1::2] << 4)
    st["scales"][_scale_at(slots, bits.shape[1] // 4)] = bits
    st["row_scale"][slots] = g


def _values(code):
    """What the codes stand for, float32."""
    m = (code & 7).float()
    v = torch.where(m < 5, 0.5 * m, torch.where(m < 6, 3.0, 2.0 * m - 8.0))
    return torch.where(code >= 8, -v, v)


def _get(st, slots):
    """Rows in units of g (float32 [n, dp], exact) and g [n]."""
    byte = st["codes"][slots]
    code = torch.stack((byte & 15, byte >> 4), 2).flatten(1)
    dp, block = code.shape[1], BLOCK[st["format"]]
    bits = st["scales"][_scale_at(slots, dp // block // 4)]
    if st["format"] == "mx":
        s = torch.ldexp(torch.ones(bits.shape, dtype=torch.float64, device=bits.device), bits.int() - 127)
        s = s.float()
    else:
        s = bits.view(torch.float8_e4m3fn).float()
    v = _values(code).view(len(slots), dp // block, block) * s[:, :, None]
    return v.view(len(slots), dp), st["row_scale"][slots]


def _plain_write(st):
    code, _, bits, g = _quantise(st["src"], st["format"])
    _put(st, st["slots"], code, bits, g)
    v, g = _get(st, st["slots"])
    return (v[:, :st["dim"]] * g[:, None]).to(st["out"])


def _plain_scores(st):
    code, scale, _, gq = _quantise(st["q"], st["format"])
    q = _values(code).view(*scale.shape, -1) * scale[:, :, None]
    v, g = _get(st, st["all"])
    s = (q.flatten(1) @ v.T) * g * gq[:, None]
    return torch.where(torch.isnan(g) | torch.isnan(gq)[:, None], -math.inf, s).to(st["out"])


def _plain_knn(st):
    code, scale, _, gq = _quantise(st["q"], st["format"])
    q = _values(code).view(*scale.shape, -1) * scale[:, :, None]
    v, g = _get(st, st["all"])
    s = q.flatten(1).double() @ v.double().T  # in 64 bits: neighbours' ranks hang on the last ones
    s = (s.mul_(g.double()).mul_(gq.double()[:, None])).float()
    s = torch.where(torch.isnan(s), -math.inf, s + 0.0)
    b = s.view(torch.int32).long()
    key = torch.where(b < 0, -(b & 0x7FFFFFFF), b) * 2 ** 32 - st["all"]  # (score, lowest slot)
    k = min(st["k"], len(st["all"]))
    ids = torch.topk(key, k, 1).indices
    out = s.gather(1, ids)
    ids = torch.where(out > -math.inf, ids, -1).int()
    pad = (0, st["k"] - k)
    return (torch.nn.functional.pad(ids, pad, value=-1),
            torch.nn.functional.pad(out, pad, value=-math.inf))


# ------------------------------------------------------------------ inputs --
def _mixture(n, dim, gen, dev, centres):
    """Unit rows around common centres, as embeddings of related documents lie."""
    at = torch.randint(len(centres), (n,), generator=gen, device=dev)
    x = torch.randn((n, dim), generator=gen, device=dev).mul_(0.3).add_(centres[at])
    return x.div_(x.norm(dim=1, keepdim=True))


def _store(x, fmt, slots):
    n, dp = len(x), _pad_dim(x.shape[1])
    atoms = dp // BLOCK[fmt] // 4
    dev = x.device
    st = {"format": fmt, "dim": x.shape[1],
          "codes": torch.zeros((slots, dp // 2), dtype=torch.uint8, device=dev),
          "scales": torch.zeros(-(-slots // 128) * atoms * 512, dtype=torch.uint8, device=dev),
          "row_scale": torch.full((slots,), math.nan, device=dev),
          "norm_max": torch.zeros(1, device=dev),
          "claim": torch.zeros(slots, dtype=torch.int32, device=dev)}
    for a in range(0, n, 65536):
        part = x[a:a + 65536]
        code, scale, bits, g = _quantise(part, fmt)
        _put(st, torch.arange(a, a + len(part), device=dev), code, bits, g)
        bound = 6.1 * g * (scale.square().sum(1) * BLOCK[fmt]).sqrt()
        st["norm_max"] = torch.maximum(st["norm_max"], bound.nan_to_num().amax())
    return st


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dim, typ = case["dim"], TYPES[case["type"]]
    centres = torch.randn((min(1024, max(4, (case.get("n") or case["rows"]) // 16)), dim),
                          generator=gen, device=dev)
    if case["op"] == "write":
        n, slots = case["rows"], case["slots"]
        st = _store(torch.zeros((0, dim), device=dev), case["format"], slots)
        wide = torch.empty((n, dim + case["pad"]), dtype=typ, device=dev)
        wide[:, :dim] = _mixture(n, dim, gen, dev, centres)
        st["src"] = wide[:, :dim]
        st["slots"] = torch.randperm(slots, generator=gen, device=dev)[:n]
        st["out"] = TYPES[case["out"]]
    else:
        st = _store(_mixture(case["n"], dim, gen, dev, centres), case["format"], case["n"])
        st["q"] = _mixture(case["nq"], dim, gen, dev, centres).to(typ)
        st["all"] = torch.arange(case["n"], device=dev)
        if case["op"] == "scores":
            st["out"] = TYPES[case["out"]]
        else:
            st["k"] = case["k"]
    st["op"] = case["op"]
    return st


# --------------------------------------------------------------------- run --
@functools.lru_cache(None)
def _context():
    import pion_b200
    return pion_b200.Context(0)


def _own(st):
    import pion_b200
    rows = pion_b200.FP4Rows(len(st["codes"]), st["dim"], st["format"], codes=st["codes"],
                             scales=st["scales"], row_scale=st["row_scale"],
                             norm_max=st["norm_max"], claim=st["claim"])
    if st["op"] == "write":
        rows.write(_context(), st["src"], slots=st["slots"])
        return rows.read(_context(), slots=st["slots"], dtype=st["out"])
    if st["op"] == "scores":
        return pion_b200.fp4_scores(_context(), rows, st["q"], dtype=st["out"])
    return pion_b200.FlatFP4Index(_context(), rows).search(st["q"], st["k"])


def run(state):
    if own:
        return _own(state)
    return {"write": _plain_write, "scores": _plain_scores, "knn": _plain_knn}[state["op"]](state)


# -------------------------------------------------------------------- work --
def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    dim = case["dim"]
    row = dim / 2 + dim / BLOCK[case["format"]] + 4
    if case["op"] == "write":
        n = case["rows"]
        return {"bytes": n * (dim * (size[case["type"]] + size[case["out"]]) + 2 * row + 16),
                "flops": 2 * n * dim}
    n, nq = case["n"], case["nq"]
    out = nq * n * size[case["out"]] if case["op"] == "scores" else nq * min(case["k"], n) * 8
    return {"bytes": n * row + nq * dim * size[case["type"]] + out, "flops": 2 * n * nq * dim}


# ------------------------------------------------------------------- exact --
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_rows(x, fmt):
    """Rows quantised by the definition, in float64: (rows in units of g, g)."""
    x = x.double()
    n, dim = x.shape
    block = BLOCK[fmt]
    blocks = torch.zeros((n, -(-dim // block) * block), dtype=torch.float64, device=x.device)
    blocks[:, :dim] = x
    blocks = blocks.view(n, -1, block)
    top = blocks.abs().max(2).values
    if fmt == "mx":
        s = torch.where(top > 0, torch.exp2(torch.floor(torch.log2(top.clamp(min=1e-300))) - 2), 1.0)
        g = torch.ones(n, dtype=torch.float64, device=x.device)
        unit = s
    else:
        g = (top.max(1).values / torch.full((), 2688.0, dtype=torch.float64, device=x.device)).float().double()
        h = (6.0 * g).float().double()
        t = top / h[:, None]
        q = 2.0 ** (torch.floor(torch.log2(t.clamp(min=2.0 ** -6))) - 3)
        s = ((t / q).round() * q).clamp(max=448.0)
        unit = (s * g[:, None]).float().double()
    grid = torch.tensor(_GRID, dtype=torch.float64, device=x.device)
    y = blocks.abs() / unit.clamp(min=1e-300)[:, :, None]
    low = (torch.bucketize(y, grid, right=True) - 1).clamp(max=6)
    low = torch.where(y >= 6.0, 6, low)
    a, b = grid[low], grid[low + 1]
    mid = 0.5 * (a + b)
    up = (y > mid) | ((y == mid) & (low % 2 == 1))
    v = torch.where(up, b, a).copysign(blocks) * s[:, :, None]
    v = torch.where(unit[:, :, None] > 0, v, 0.0)
    return v.view(n, -1)[:, :dim], g


def _exact_store(st):
    lut = torch.tensor(_GRID + tuple(-v for v in _GRID), dtype=torch.float64, device=st["codes"].device)
    n, dim, block = len(st["codes"]), st["dim"], BLOCK[st["format"]]
    atoms = st["codes"].shape[1] * 2 // block // 4
    tiles = st["scales"].view(-1, atoms, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, atoms * 4)[:n]
    byte = torch.arange(256, device=tiles.device)
    if st["format"] == "mx":
        table = torch.exp2(byte.double() - 127)
    else:
        e, m = (byte >> 3).double(), (byte & 7).double()
        table = torch.where(e > 0, (8 + m) * 2.0 ** (e - 10), m * 2.0 ** -9)
    for a in range(0, n, 32768):
        c = st["codes"][a:a + 32768].long()
        v = torch.empty((len(c), 2 * c.shape[1]), dtype=torch.float64, device=c.device)
        v[:, 0::2], v[:, 1::2] = lut[c & 15], lut[c >> 4]
        v *= table[tiles[a:a + 32768].long()].repeat_interleave(block, 1)
        yield a, v[:, :dim], st["row_scale"][a:a + 32768].double()


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "write":
        parts = []
        for a in range(0, case["rows"], 65536):
            v, g = _exact_rows(st["src"][a:a + 65536], st["format"])
            parts.append(v * g[:, None])
        return torch.cat(parts)
    q, gq = _exact_rows(st["q"], st["format"])
    if case["op"] == "scores":
        return torch.cat([(q @ v.T) * g * gq[:, None] for _, v, g in _exact_store(st)], 1)
    best = None
    for a, v, g in _exact_store(st):
        s = (q @ v.T) * g * gq[:, None]
        s = torch.cat([best, s], 1) if best is not None else s
        best = torch.topk(s, min(case["k"], s.shape[1]), 1).values
    best = torch.nn.functional.pad(best, (0, case["k"] - best.shape[1]), value=-math.inf)
    return None, best  # the ids have to be equal, and have no rounding to speak of
