"""Searches built from the kernel's own geometry (tiles of 256 rows, of which 64, or for more than 64
queries 32, evenly spaced ones give the first thresholds), and compositions of the 4-bit calls."""
import ctypes

import numpy as np
import pytest
import torch

import fp4_plain as plain

pytestmark = pytest.mark.gpu

TILE, KEPT = 256, 4096   # rows of a tile; candidates kept per query


def geometry(n, nq):
    """(tile step of the sample, of the first part searched) of a search that samples."""
    tiles, samples = -(-n // TILE), 64 if nq <= 64 else 32
    assert nq * n > 2 ** 22 and tiles > samples      # else every row's score is written
    ratio, stages = tiles / samples, 1
    while nq > 64 and int(np.ceil(ratio ** (1 / stages))) > 12:
        stages += 1
    grow = max(2, int(np.ceil(ratio ** (1 / stages))))
    return tiles // samples, grow ** (stages - 1)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("n,nq,also_first", [(70000, 64, False), (70100, 100, False),
                                             (200000, 100, False), (200000, 100, True)])
def test_a_sample_that_misses_the_best_rows(ctx, fmt, n, nq, also_first):
    """Every sampled tile is poor (and every one of the first part), the rest rich: far more rows
    reach the sample's threshold than are kept, and the queries are answered by the scan."""
    import pion_b200
    rng = np.random.default_rng(n + nq)
    step, first = geometry(n, nq)
    samples = 64 if nq <= 64 else 32
    tile = np.arange(n) // TILE
    poor = (tile % step == 0) & (tile < step * samples)
    if also_first:
        assert first > 1
        poor |= tile % first == 0
    base = rng.standard_normal(64)
    x = rng.standard_normal((n, 64)) * 0.1
    x[~poor] += base
    q = base + 0.3 * rng.standard_normal((nq, 64))
    q[::7] = -q[::7]                                  # for some the poor ones are the best
    x, q = x.astype(np.float32), q.astype(np.float32)
    want, _ = plain.products(q.astype(np.float64), x.astype(np.float64), fmt)
    sampled = np.flatnonzero((tile % step == 0) & (tile < step * samples))
    assert poor[sampled].all() and len(sampled) == samples * TILE
    kth = np.sort(want[:, sampled], axis=1)[:, -10]
    over = (want > kth[:, None]).sum(1)
    assert (np.delete(over, np.s_[::7]) > KEPT).all()
    rows = pion_b200.quantize_rows_fp4(ctx, torch.from_numpy(x).cuda(), fmt)
    ids, sc = pion_b200.FlatFP4Index(ctx, rows).search(torch.from_numpy(q).cuda(), 10)
    torch.cuda.synchronize()
    ctx.sync()
    wi, wv = plain.best(want, 10)
    assert np.array_equal(ids.cpu().numpy(), wi)
    assert np.array_equal(sc.cpu().numpy().view(np.uint32), wv.view(np.uint32))


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_shards_merge_to_one_stores_answer(ctx, fmt):
    """Row shards searched each for itself, merged by merge_topk: ids and scores of the one store,
    with ties across shards, empty slots, and a shard of fewer than k rows."""
    import pion_b200
    rng = np.random.default_rng(12)
    n, k = 9000, 20
    x = rng.standard_normal((n, 100)).astype(np.float32)
    x[[10, 4000, 4001, 8995]] = x[5000]
    x[rng.integers(0, n, 400)] = np.nan
    q = rng.standard_normal((37, 100)).astype(np.float32)
    q[3] = x[5000]
    q[4] = 0
    tx, tq = torch.from_numpy(x).cuda(), torch.from_numpy(q).cuda()
    whole = pion_b200.FlatFP4Index(ctx, pion_b200.quantize_rows_fp4(ctx, tx, fmt)).search(tq, k)
    parts = []
    for a, b in ((0, 4001), (4001, 8990), (8990, 9000)):
        rows = pion_b200.quantize_rows_fp4(ctx, tx[a:b], fmt)
        parts.append(pion_b200.FlatFP4Index(ctx, rows, id_base=a).search(tq, k))
    torch.cuda.synchronize()
    for major in (False, True):
        ids = torch.stack([p[0] for p in parts], 0 if major else 1).contiguous()
        sc = torch.stack([p[1] for p in parts], 0 if major else 1).contiguous()
        got = pion_b200.merge_topk(ctx, sc, ids, k, lists_major=major)
        torch.cuda.synchronize()
        ctx.sync()
        assert torch.equal(got[0], whole[0]) and torch.equal(got[1], whole[1])


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("type_,dtype", [(0, np.float32), (2, np.float16)])
def test_read_into_host_memory(ctx, fmt, type_, dtype):
    """pion_v_b200_fp4_read with host memory: slots and ranges, rows inside a wider buffer whose
    other elements stay as they were, and its refusals."""
    import pion_b200
    from pion_b200 import _lib
    rng = np.random.default_rng(7)
    n, dim, stride = 300, 77, 81
    rows = pion_b200.quantize_rows_fp4(ctx, rng.standard_normal((n, dim)).astype(np.float32), fmt)
    torch.cuda.synchronize()
    slots = rng.integers(0, n, 50).astype(np.int64)
    want = rows.read(ctx, dtype=torch.float32 if type_ == 0 else torch.float16).cpu().numpy()
    out = np.full((50, stride), 7, dtype)

    def read(ps, start, count, dst=out, st=stride):
        return ctx.lib.pion_v_b200_fp4_read(ctx.h, rows._ref(ctx), ps, start, count,
                                            dst.ctypes.data_as(ctypes.c_void_p), type_, st,
                                            _lib.MEM_HOST, None)

    assert read(slots.ctypes.data_as(ctypes.c_void_p), 0, 50) == 0
    assert np.array_equal(out[:, :dim], want[slots]) and (out[:, dim:] == 7).all()
    assert read(None, 250, 50) == 0
    assert np.array_equal(out[:, :dim], want[250:]) and (out[:, dim:] == 7).all()
    assert read(None, 3, 1, st=dim) == 0
    assert np.array_equal(out[0, :dim], want[3])
    out[:] = 7
    for bad in ([-1], [n], [0, 2 ** 40]):
        ps = np.array(bad, np.int64)
        assert read(ps.ctypes.data_as(ctypes.c_void_p), 0, len(bad)) == _lib.EINVAL
    assert read(None, 251, 50) == _lib.EINVAL and read(None, -1, 2) == _lib.EINVAL
    assert read(None, 0, 2, st=dim - 1) == _lib.EINVAL
    assert read(None, 0, 0) == 0
    assert (out == 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scores_of_more_than_two_to_31(ctx, dtype):
    """A score matrix of 2.3e9 elements: its last rows and columns are those of small calls."""
    import pion_b200
    n, nq, dim = 2_100_003, 1100, 128
    assert n * nq > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((n, dim), device="cuda", generator=g)
    q = torch.randn((nq, dim), device="cuda", generator=g)
    rows = pion_b200.quantize_rows_fp4(ctx, x, "nv")
    tail = pion_b200.quantize_rows_fp4(ctx, x[n - 515:], "nv")
    out = pion_b200.fp4_scores(ctx, rows, q, dtype=dtype)
    last = pion_b200.fp4_scores(ctx, tail, q, dtype=dtype)
    some = pion_b200.fp4_scores(ctx, rows, q[-3:], dtype=dtype)
    torch.cuda.synchronize()
    ctx.sync()
    assert torch.equal(out[:, n - 515:], last)
    assert torch.equal(out[-3:], some)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("dim", [64, 128, 1536, 8192])
def test_error_bound_where_products_are_cut_off(ctx, fmt, dim):
    """The search's premise, |approximate - exact| <= (dp / 64 + 8) 2^-22 |q| |v|, where an adder that
    cuts off at its largest term loses most: one large product, all others just below its last bits,
    of one sign, in the same step and in later ones."""
    import pion_b200
    block = plain.BLOCK[fmt]
    xs, qs = [], []
    for gap in range(8, 17):                 # small products are 2^-2gap of the large one
        for extra in (0, 1):
            for big, small in ((6.0, 6.0), (4.0, 6.0), (4.0, 1.0), (6.0, 1.5), (4.0, 3.0), (1.0, 6.0)):
                for sign in (1.0, -1.0):
                    x = np.full(dim, small * 2.0 ** (-gap - extra))
                    q = np.full(dim, small * 2.0 ** -gap)
                    x[:block], q[:block] = 0, 0
                    x[0], q[0] = big, sign * big
                    xs.append(x), qs.append(q)
                    x, q = x.copy(), q.copy()          # the large one in the last block
                    x[[0, dim - 1]], q[[0, dim - 1]] = x[[dim - 1, 0]], q[[dim - 1, 0]]
                    x[dim - block:dim - 1] = q[dim - block:dim - 1] = 0
                    x[1:block], q[1:block] = x[0], q[0]
                    xs.append(x), qs.append(q)
    x, q = np.float32(xs), np.float32(qs)
    rows = pion_b200.quantize_rows_fp4(ctx, torch.from_numpy(x).cuda(), fmt)
    got = pion_b200.fp4_scores(ctx, rows, torch.from_numpy(q).cuda())
    torch.cuda.synchronize()
    ctx.sync()
    want, _ = plain.products(q.astype(np.float64), x.astype(np.float64), fmt)

    def norms(v):
        c, b, g = plain.quantise(v.astype(np.float64), fmt)
        return np.linalg.norm(plain.values(c, b, fmt), axis=1) * g

    off = (np.abs(got.double().cpu().numpy() - want) / (norms(q)[:, None] * norms(x))).max()
    print(f"{fmt} dim {dim}: largest error {off:.3g} |q||v| = 2^{np.log2(off + 1e-30):.1f}")
    assert off <= (plain.pad_dim(dim) / 64 + 8) * 2.0 ** -22
