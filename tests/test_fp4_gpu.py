"""Microscaled 4-bit rows on the GPU against their definition in float64 (tests/fp4_plain.py).

What is compared how: codes, scale bytes, row scales and float32 read-backs bit for bit;
16-bit read-backs and scores within half a step of the output type (plus, for scores, the
bound of a float32 sum of dp terms in any order, rounded or truncated: dp 2^-23 times the sum
of the terms' magnitudes); ids and scores of a search bit for bit."""
import numpy as np
import pytest
import torch

import fp4_plain as plain
from pion_b200.workloads import mixture_np

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# smallest subnormal step of each type
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}


def half_step(dtype, ref):
    return torch.finfo(TYPES[dtype]).eps / 2 * np.abs(ref) + TINY[dtype] / 2


def typed(x, dtype):
    """x as a CUDA tensor of a type, and its exact values in float64."""
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(TYPES[dtype])
    return t.cuda(), t.double().numpy()


def rows_np(n, dim, seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, dim)) * np.exp2(rng.integers(-6, 7, (n, 1)))
    return x * np.exp(rng.standard_normal((n, dim)) * 0.5)


def finish(ctx):
    """Waits for torch's streams, then takes what the calls' kernels have reported."""
    torch.cuda.synchronize()
    ctx.sync()


def unpack(rows):
    c = rows.codes.cpu().numpy()
    return np.stack((c & 15, c >> 4), 2).reshape(len(c), -1)


def check_store(rows, slots, x, fmt):
    """The store's slots hold exactly the rows x (a code of minus zero counts as zero)."""
    codes, bits, g = plain.quantise(x, fmt)
    got = unpack(rows)[slots]
    got = np.where(got == 8, 0, got)
    live = ~np.isnan(g)
    assert np.array_equal(got[live], np.where(codes == 8, 0, codes)[live])
    atoms = rows.scales.numel() // (-(-rows.n_rows // 128) * 512)
    sb = plain.row_scales(rows.scales.cpu().numpy(), rows.n_rows, atoms)[slots]
    assert np.array_equal(sb[live], bits[live])
    rs = rows.row_scale.cpu().numpy()[slots]
    assert np.array_equal(rs.view(np.uint32)[live], g.view(np.uint32)[live])
    assert np.isnan(rs[~live]).all()
    norms = np.sqrt((plain.values(codes, bits, fmt)[live] ** 2).sum(1)) * g[live]
    assert float(rows.norm_max) >= norms.max(initial=0.0)
    return codes, bits, g


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,dim,pad", [(1, 1, 0), (3, 15, 1), (9, 16, 0), (130, 33, 3),
                                       (64, 128, 8), (257, 384, 0), (20, 777, 7), (33, 1536, 0),
                                       (5, 2049, 0), (2, 8192, 0), (1100, 1536, 0),
                                       (1030, 1900, 0), (1027, 4096, 0), (1025, 5000, 3),
                                       (1051, 600, 1), (1026, 768, 0),
                                       (1029, 1024, 8), (1040, 2048, 0), (1033, 256, 0)])
def test_write_and_read(ctx, fmt, dtype, n, dim, pad):
    import pion_b200
    x = rows_np(n, dim, n * dim + pad)
    x[0, :] = np.abs(x[0, :])
    wide, exact = typed(np.pad(x, ((0, 0), (0, pad)), constant_values=np.nan), dtype)
    src, exact = wide[:, :dim], exact[:, :dim]
    rows = pion_b200.FP4Rows(n + 5, dim, fmt)
    slots = np.random.default_rng(1).permutation(n + 5)[:n]
    rows.write(ctx, src, slots=torch.from_numpy(slots).cuda())
    finish(ctx)
    codes, bits, g = check_store(rows, slots, exact, fmt)
    rest = np.setdiff1d(np.arange(n + 5), slots)
    assert np.isnan(rows.row_scale.cpu().numpy()[rest]).all()
    assert not unpack(rows)[rest].any()
    assert not rows.claim.any()
    want = plain.values(codes, bits, fmt)[:, :dim] * g[:, None].astype(np.float64)
    for out in TYPES:
        got = rows.read(ctx, slots=slots, dtype=TYPES[out]).double().cpu().numpy()
        if out == "f32":
            assert np.array_equal(got, want.astype(np.float32).astype(np.float64))
        else:
            fits = np.abs(want) <= torch.finfo(TYPES[out]).max
            # rounded through float32: half a step of the type and half of one of float32
            tol = half_step(out, want) + half_step("f32", want)
            assert (np.abs(got - want) <= tol)[fits].all()
    assert np.isnan(rows.read(ctx, slots=rest).cpu().numpy()).all()


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_ties_and_borders(ctx, fmt):
    """Small integers and halves fall on the borders between codes and between scales."""
    import pion_b200
    rng = np.random.default_rng(3)
    x = rng.integers(-48, 49, (4000, 96)).astype(np.float64) / 8
    x[::2] *= np.exp2(rng.integers(-40, 40, (2000, 1)))
    x[1::4] = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], (1000, 96))
    x[1::4, 0] = 6.0 * 448 / rng.choice([1, 2, 4, 8, 16], 1000)
    x[2::4, ::16] = 2688.0 * rng.integers(1, 9, (1000, 6)) / 8
    t, exact = typed(x, "f32")
    # neighbours of the borders, one step up and down
    up = torch.nextafter(t, torch.full_like(t, np.inf))
    down = torch.nextafter(t, torch.full_like(t, -np.inf))
    for v in (t, up, down):
        rows = pion_b200.quantize_rows_fp4(ctx, v, fmt)
        check_store(rows, np.arange(4000), v.double().cpu().numpy(), fmt)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_extreme_rows(ctx, fmt):
    """Zero rows, zero blocks, the largest and the smallest magnitudes, NaN and infinities."""
    import pion_b200
    x = rows_np(16, 200, 5).astype(np.float32)
    x[0] = 0
    x[1, :64] = 0
    x[2] = np.float32(3.0e38)
    x[3] *= np.float32(2.0 ** -120)
    x[4] = np.float32(2.0 ** -149)
    x[5] = 0
    x[5, 7] = np.float32(2.0 ** -126)
    x[6, 199] = np.nan
    x[7, 0] = np.inf
    x[8, 100] = -np.inf
    x[9] *= np.float32(2.0 ** -99) / np.abs(x[9]).max()
    x[10, 3] = np.finfo(np.float32).max
    x[11, 16:] *= np.float32(2.0 ** -30)
    x[12] = np.float32(2.0 ** -100)
    x[13] = np.nextafter(np.float32(2.0 ** -100), np.float32(0))
    rows = pion_b200.quantize_rows_fp4(ctx, torch.from_numpy(x).cuda(), fmt)
    codes, bits, g = check_store(rows, np.arange(16), x, fmt)
    want = plain.values(codes, bits, fmt)[:, :200] * g[:, None].astype(np.float64)
    with np.errstate(over="ignore"):
        want = want.astype(np.float32)
    got = rows.read(ctx).cpu().numpy()
    live = ~np.isnan(g)
    assert np.array_equal(got[live], want[live])
    assert np.isnan(got[[6, 7, 8]]).all() and live.sum() == 13


def test_slots_repeated_skipped_and_out_of_range(ctx):
    import pion_b200
    x = rows_np(300, 64, 11)
    t, exact = typed(x, "f32")
    for on_gpu in (True, False):
        rows = pion_b200.FP4Rows(40, 64, "nv")
        slots = np.random.default_rng(2).integers(0, 20, 300)
        slots[::7] = -1
        rows.write(ctx, t if on_gpu else t.cpu(),
                   slots=torch.from_numpy(slots).cuda() if on_gpu else slots)
        finish(ctx)
        last = {s: i for i, s in enumerate(slots.tolist()) if s >= 0}
        at = np.array(sorted(last))
        check_store(rows, at, exact[[last[s] for s in at.tolist()]], "nv")
        assert torch.isnan(rows.row_scale[20:]).all() and not rows.claim.any()
    before = [b.clone() for b in (rows.codes, rows.scales, rows.row_scale)]
    slots = np.full(300, 40)
    with pytest.raises(pion_b200.PionError):
        rows.write(ctx, x.astype(np.float32), slots=slots)       # host: refused
    rows.write(ctx, t, slots=torch.from_numpy(slots).cuda())      # device: skipped, reported
    with pytest.raises(pion_b200.PionError) as e:
        finish(ctx)
    assert e.value.code == -1
    out = torch.full((2, 64), 5.0, device="cuda")
    rows.read(ctx, slots=torch.tensor([-1, 45]).cuda(), out=out)
    with pytest.raises(pion_b200.PionError):
        finish(ctx)
    assert (out == 5.0).all()
    for a, b in zip(before, (rows.codes, rows.scales, rows.row_scale)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    rows.clear(ctx)
    assert torch.isnan(rows.read(ctx)).all()


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("dim", [40, 1900, 4000, 5000])
def test_many_rows_for_the_same_slots(ctx, fmt, dim):
    """More rows than are written by a CTA each, most of them for a slot of a later row, one and
    two warps a row; again into the same store, whose claims were left at zero."""
    import pion_b200
    rng = np.random.default_rng(dim)
    rows = pion_b200.FP4Rows(700, dim, fmt)
    x = rows_np(1500, dim, 77)
    t, exact = typed(x, "f32")
    for _ in range(2):
        slots = rng.integers(-20, 600, 1500)
        rows.clear(ctx)
        rows.write(ctx, t, slots=torch.from_numpy(slots).cuda())
        finish(ctx)
        last = {s: i for i, s in enumerate(slots.tolist()) if s >= 0}
        at = np.array(sorted(last))
        check_store(rows, at, exact[[last[s] for s in at.tolist()]], fmt)
        rest = np.setdiff1d(np.arange(700), at)
        assert torch.isnan(rows.row_scale[torch.from_numpy(rest).cuda()]).all()
        assert not rows.claim.any()


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("n,dim,nq,types", [
    (1, 1, 1, "f32 f32"), (5, 40, 3, "bf16 f16"), (127, 128, 16, "f32 bf16"),
    (129, 200, 17, "f16 f32"), (1000, 384, 208, "f32 f32"), (700, 1536, 209, "bf16 bf16"),
    (3001, 1536, 64, "f32 f16"), (40000, 256, 2, "f32 f32"), (500, 8192, 40, "f32 f32"),
    (900, 4100, 130, "f32 f32"), (300, 64, 3000, "f32 f32"), (6000, 96, 500, "f32 bf16")])
def test_scores(ctx, fmt, n, dim, nq, types):
    import pion_b200
    tq, to = types.split()
    x, q = rows_np(n, dim, n), rows_np(nq, dim, nq + 7)
    x[n // 2] = 0
    q[nq // 2] = 0
    if n > 4:
        x[3, dim // 2] = np.nan
    if nq > 2:
        q[1, dim - 1] = np.inf
    tx, ex = typed(x, "f32")
    tq_, eq = typed(q, tq)
    rows = pion_b200.FP4Rows(n + 3, dim, fmt)
    rows.write(ctx, tx)
    want, size = plain.products(eq, ex, fmt)
    got = pion_b200.fp4_scores(ctx, rows, tq_, dtype=TYPES[to])
    finish(ctx)
    got = got.double().cpu().numpy()
    assert np.isneginf(got[:, n:]).all()
    got = got[:, :n]
    if nq > 2:
        assert np.isneginf(got[1]).all()
        keep = np.arange(nq) != 1
        got, want, size = got[keep], want[keep], size[keep]
    if n > 4:
        assert np.isneginf(got[:, 3]).all()
        keep = np.arange(n) != 3
        got, want, size = got[:, keep], want[:, keep], size[:, keep]
    fits = np.abs(want) < torch.finfo(TYPES[to]).max / 2
    tol = half_step(to, want) + plain.pad_dim(dim) * 2.0 ** -23 * size + half_step("f32", want) * 2
    assert (np.abs(got - want) <= tol * (1 + 2.0 ** -8))[fits].all()
    # part of the rows, into a wider buffer whose other columns stay as they were
    m = max(1, n // 2)
    wide = torch.full((nq, m + 5), 7.0, dtype=TYPES[to], device="cuda")
    pion_b200.fp4_scores(ctx, rows, tq_, n_rows=m, out=wide[:, :m])
    finish(ctx)
    full = pion_b200.fp4_scores(ctx, rows, tq_, dtype=TYPES[to])
    assert torch.equal(wide[:, :m], full[:, :m]) and (wide[:, m:] == 7.0).all()


def test_scores_error_bound_of_the_search(ctx):
    """The search's premise: an approximate score is within (dp / 64 + 8) 2^-22 |q| |v| of the
    exact one, also for rows whose blocks span many magnitudes."""
    import pion_b200
    rng = np.random.default_rng(8)
    for fmt in ("mx", "nv"):
        for dim in (64, 1536, 8192):
            x = rng.standard_normal((2000, dim)) * np.exp2(rng.integers(-8, 9, (2000, dim)))
            q = rng.standard_normal((64, dim)) * np.exp2(rng.integers(-8, 9, (64, dim)))
            x[:64] = q + 0.01 * rng.standard_normal((64, dim))
            tx, ex = typed(x, "f32")
            tq, eq = typed(q, "f32")
            rows = pion_b200.quantize_rows_fp4(ctx, tx, fmt)
            got = pion_b200.fp4_scores(ctx, rows, tq).double().cpu().numpy()
            want, _ = plain.products(eq, ex, fmt)
            qc, qb, qg = plain.quantise(eq, fmt)
            rc, rb, rg = plain.quantise(ex, fmt)
            nq = np.linalg.norm(plain.values(qc, qb, fmt), axis=1) * qg
            nr = np.linalg.norm(plain.values(rc, rb, fmt), axis=1) * rg
            off = (np.abs(got - want) / (nq[:, None] * nr)).max()
            print(f"{fmt} dim {dim}: largest error {off:.3g} |q||v| = 2^{np.log2(off + 1e-30):.1f}")
            assert off <= (plain.pad_dim(dim) / 64 + 8) * 2.0 ** -22


def check_knn(ctx, rows, q, exact_q, exact_x, fmt, k, n_rows=None, id_base=0):
    import pion_b200
    ids, sc = pion_b200.FlatFP4Index(ctx, rows, id_base=id_base).search(q, k, n_rows=n_rows)
    finish(ctx)
    n = len(exact_x) if n_rows is None else n_rows
    want, _ = plain.products(exact_q, exact_x[:n], fmt)
    wi, wv = plain.best(want, k)
    wi = np.where(wi >= 0, wi + id_base, -1)
    if torch.is_tensor(ids):
        ids, sc = ids.cpu().numpy(), sc.cpu().numpy()
    assert np.array_equal(ids, wi)
    assert np.array_equal(sc.view(np.uint32), wv.view(np.uint32))


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("n,dim,nq,k,dtype", [
    (1, 16, 1, 1, "f32"), (5, 100, 3, 10, "f32"), (1000, 1536, 1, 10, "bf16"),
    (8192, 128, 33, 64, "f32"), (8193, 130, 5, 256, "f16"), (8320, 64, 3, 1, "f32"),
    (20011, 384, 209, 10, "f32"), (60000, 256, 16, 256, "f32"), (150000, 96, 7, 100, "f32"),
    (300003, 40, 20, 10, "f32"), (90001, 64, 60, 256, "f32"), (70000, 100, 150, 33, "bf16"),
    (24577, 200, 1, 10, "f32"), (24576, 200, 4, 1, "f32")])
def test_knn(ctx, fmt, n, dim, nq, k, dtype):
    import pion_b200
    x, q = mixture_np(n, dim, max(1, n // 200), seed=n + k, n_queries=nq)
    tx, ex = typed(x, "f32")
    tq, eq = typed(q, dtype)
    rows = pion_b200.quantize_rows_fp4(ctx, tx, fmt)
    check_knn(ctx, rows, tq, eq, ex, fmt, k)


def test_knn_ties_empty_rows_and_odd_queries(ctx):
    import pion_b200
    rng = np.random.default_rng(4)
    for fmt in ("mx", "nv"):
        for n in (3000, 30000):
            x, q = mixture_np(n, 160, 40, seed=n, n_queries=8)
            x, q = x.copy(), q.copy()
            x[rng.integers(0, n, 300)] = x[5]            # equal scores: lowest id first
            x[rng.integers(0, n, 200)] = np.nan          # empty slots
            x[rng.integers(0, n, 200)] = 0
            q[0], q[1], q[2, 3], q[3] = x[5], 0, np.nan, -q[3]
            tx, ex = typed(x, "f32")
            tq, eq = typed(q, "f32")
            rows = pion_b200.quantize_rows_fp4(ctx, tx, fmt)
            for k in (1, 10, 200):
                check_knn(ctx, rows, tq, eq, ex, fmt, k)
            check_knn(ctx, rows, tq, eq, ex, fmt, 10, n_rows=n // 3, id_base=1000)
            check_knn(ctx, rows, tq, eq, ex, fmt, 10, n_rows=7)
    rows = pion_b200.FP4Rows(20000, 160, "nv")           # nothing but empty slots
    ids, sc = pion_b200.FlatFP4Index(ctx, rows).search(tq, 5)
    assert (ids == -1).all() and torch.isneginf(sc).all()
    rows.write(ctx, tx[:1], start=19999)                  # one row at the end
    ids, sc = pion_b200.FlatFP4Index(ctx, rows).search(tq[:1], 5)
    assert ids.tolist() == [[19999, -1, -1, -1, -1]]
    ids, sc = pion_b200.FlatFP4Index(ctx, rows).search(tq[:1], 5, n_rows=0)
    assert (ids == -1).all()


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_knn_overflowing_candidates(ctx, fmt):
    """More rows reach the threshold than are kept: all equal, ascending along the index, or
    of norms whose products leave float32."""
    import pion_b200
    rng = np.random.default_rng(6)
    x = np.repeat(rng.standard_normal((1, 64)), 12000, 0)
    q = np.concatenate([x[:1], -x[:1], rng.standard_normal((1, 64))])
    tx, ex = typed(x, "f32")
    tq, eq = typed(q, "f32")
    rows = pion_b200.quantize_rows_fp4(ctx, tx, fmt)
    check_knn(ctx, rows, tq, eq, ex, fmt, 20)
    # every sampled tile of 128 rows is poor, the rest rich
    n = 40000
    x = rng.standard_normal((n, 64)) * 0.1
    tiles = -(-n // 128)
    rich = (np.arange(n) // 128) % (tiles // 64) != 0
    x[rich] += q[2]
    tx, ex = typed(x, "f32")
    rows = pion_b200.quantize_rows_fp4(ctx, tx, fmt)
    check_knn(ctx, rows, tq, eq, ex, fmt, 10)
    many = np.repeat(eq, 50, 0)                           # the same with sampled thresholds
    check_knn(ctx, rows, typed(many, "f32")[0], many, ex, fmt, 10)
    x[n // 2:] = x[5]                                     # a chunk of equal rows
    tx, ex = typed(x, "f32")
    rows = pion_b200.quantize_rows_fp4(ctx, tx, fmt)
    near = ex[5:6]
    check_knn(ctx, rows, typed(near, "f32")[0], near, ex, fmt, 10)
    x = rng.standard_normal((10000, 64)) * 2.0 ** 63
    tx, ex = typed(x, "f32")
    tq, eq = typed(q * 2.0 ** 62, "f32")
    rows = pion_b200.quantize_rows_fp4(ctx, tx, fmt)
    check_knn(ctx, rows, tq, eq, ex, fmt, 10)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("n,nq", [(9000, 3), (40000, 3), (40000, 150)])
@pytest.mark.parametrize("row_exp,q_exp", [(114, -12), (-70, 110), (-95, 0), (100, -99)])
def test_knn_far_magnitudes(ctx, fmt, n, nq, row_exp, q_exp):
    """Scores inside float32 whose factors are far apart: the product with the row's g alone
    may leave it."""
    import pion_b200
    rng = np.random.default_rng(n + nq)
    tx, ex = typed(rng.standard_normal((n, 64)) * 2.0 ** row_exp, "f32")
    tq, eq = typed(rng.standard_normal((nq, 64)) * 2.0 ** q_exp, "f32")
    rows = pion_b200.quantize_rows_fp4(ctx, tx, fmt)
    check_knn(ctx, rows, tq, eq, ex, fmt, 10)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("row_exp,q_exp", [(0, 0), (-115, 50), (-120, 55), (-120, 100),
                                           (50, -115), (80, -90)])
def test_knn_ties_that_float32_sums_tell_apart(ctx, fmt, row_exp, q_exp):
    """Rows made of the same 16 chunks in another order: equal scores, whose float32 sums
    differ.  The lowest ids are the best, at every magnitude of rows and queries."""
    import pion_b200
    rng = np.random.default_rng(41)
    n, tied = 17000, 100
    chunks = rng.standard_normal((16, 64)) * 2.0 ** rng.integers(0, 28, (16, 1))
    piece = rng.standard_normal(64)
    chunks *= np.sign(chunks @ piece)[:, None]
    x = np.zeros((n, 1024), np.float32)
    x[:, :64] = rng.standard_normal((n, 64))
    for i in rng.choice(n, tied, replace=False):
        x[i] = chunks[rng.permutation(16)].reshape(-1)
    tx, ex = typed(x * 2.0 ** row_exp, "f32")
    for nq in (2, 130):
        q = np.tile(piece, (nq, 16)) * 2.0 ** (q_exp + np.arange(nq) % 2)[:, None]
        tq, eq = typed(q, "f32")
        rows = pion_b200.quantize_rows_fp4(ctx, tx, fmt)
        check_knn(ctx, rows, tq, eq, ex, fmt, 10)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_knn_beside_a_long_row(ctx, fmt):
    """One row many times longer than the rest widens every query's margin."""
    import pion_b200
    rng = np.random.default_rng(23)
    x = rng.standard_normal((40000, 64))
    for factor in (30.0, 1e4, 1e8):
        y = x.copy()
        y[777] *= factor
        tx, ex = typed(y, "f32")
        rows = pion_b200.quantize_rows_fp4(ctx, tx, fmt)
        for nq in (3, 150):
            tq, eq = typed(rng.standard_normal((nq, 64)), "f32")
            check_knn(ctx, rows, tq, eq, ex, fmt, 10)


def test_many_overflowing_queries(ctx):
    """More flagged queries than the rescue's CTAs, and fewer; beside ordinary ones."""
    import pion_b200
    rng = np.random.default_rng(16)
    x = rng.standard_normal((9000, 48))
    x[::2] = x[0]
    tx, ex = typed(x, "f32")
    rows = pion_b200.quantize_rows_fp4(ctx, tx, "nv")
    for nq, same in ((700, 400), (90, 2), (40, 30)):
        q = rng.standard_normal((nq, 48))
        q[nq - same:] = x[0] + 0.01 * rng.standard_normal((same, 48))
        tq, eq = typed(q, "f32")
        check_knn(ctx, rows, tq, eq, ex, "nv", 33)


def test_wait_that_runs_out(ctx, monkeypatch):
    """One pair's issuer waits on a barrier that nothing arrives on: the product gives up after
    the budget, drains and reports it; the next call is right."""
    import pion_b200
    x, q = mixture_np(20000, 512, 30, seed=4, n_queries=300)
    tx, tq = torch.from_numpy(x).cuda(), torch.from_numpy(q).cuda()
    rows = pion_b200.quantize_rows_fp4(ctx, tx, "nv")
    ix = pion_b200.FlatFP4Index(ctx, rows)
    ids, sc = ix.search(tq, 10)
    full = pion_b200.fp4_scores(ctx, rows, tq)
    finish(ctx)
    ctx.set_wait_budget(1_000_000)
    try:
        for nq in (300, 1):
            monkeypatch.setenv("PION_B200_TEST_STALL", "1")
            pion_b200.fp4_scores(ctx, rows, tq[:nq])
            with pytest.raises(pion_b200.PionError) as e:
                finish(ctx)
            assert e.value.code == -11
            ix.search(tq[:nq], 10)
            with pytest.raises(pion_b200.PionError):
                finish(ctx)
            with pytest.raises(pion_b200.PionError):
                ix.search(q[:nq], 10)                    # host memory: reported by the call
            monkeypatch.delenv("PION_B200_TEST_STALL")
            again, sc2 = ix.search(tq, 10)
            assert torch.equal(again, ids) and torch.equal(sc2, sc)
            assert torch.equal(pion_b200.fp4_scores(ctx, rows, tq), full)
            finish(ctx)
    finally:
        monkeypatch.delenv("PION_B200_TEST_STALL", raising=False)
        ctx.set_wait_budget(0)


def test_refusals(ctx):
    import pion_b200
    from pion_b200 import _lib
    rows = pion_b200.FP4Rows(100, 64, "nv")
    x = torch.zeros((10, 64), device="cuda")
    ix = pion_b200.FlatFP4Index(ctx, rows)
    for bad in (lambda: rows.write(ctx, x, start=91), lambda: rows.write(ctx, x, start=-1),
                lambda: rows.read(ctx, start=95, count=6), lambda: rows.read(ctx, start=-1, count=2),
                lambda: pion_b200.fp4_scores(ctx, rows, x, n_rows=101),
                lambda: ix.search(x, 0), lambda: ix.search(x, 257), lambda: ix.search(x, 5, n_rows=101),
                lambda: pion_b200.FlatFP4Index(ctx, rows, id_base=-1).search(x, 1),
                lambda: pion_b200.FlatFP4Index(ctx, rows, id_base=2 ** 31 - 50).search(x, 1)):
        with pytest.raises(pion_b200.PionError):
            bad()
    for bad, err in ((lambda: rows.write(ctx, x[:, :63]), ValueError),
                     (lambda: rows.write(ctx, x.double()), TypeError),
                     (lambda: rows.write(ctx, x, slots=[1, 2]), ValueError),
                     (lambda: rows.write(ctx, x, slots=torch.zeros(10, device="cuda")), TypeError),
                     (lambda: rows.read(ctx, slots=[1], dtype=torch.float64), TypeError),
                     (lambda: rows.read(ctx, slots=[1], out=torch.zeros((2, 64), device="cuda")), ValueError),
                     (lambda: pion_b200.fp4_scores(ctx, rows, x, out=torch.zeros((10, 100))), ValueError),
                     (lambda: pion_b200.fp4_scores(ctx, rows, x[0]), ValueError)):
        with pytest.raises(err):
            bad()
    # a stream of its own needs a workspace; one that is too small is refused
    out = torch.empty((10, 100), device="cuda")
    wide = 2 ** 62                                        # ... and rows that span past 64 bits
    for dst, q_stride, ld in ((out, wide, 100), (out, 64, wide)):
        assert ctx.lib.pion_v_b200_fp4_scores(
            ctx.h, rows._ref(ctx), 100, x.data_ptr(), 0, q_stride, 10, dst.data_ptr(), 0, ld, None,
            0, 0, None) == _lib.EINVAL
    call = lambda ws, n: ctx.lib.pion_v_b200_fp4_scores(  # noqa: E731
        ctx.h, rows._ref(ctx), 100, x.data_ptr(), 0, 64, 10, out.data_ptr(), 0, 100, ws, n, 1, 1)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    assert call(None, 0) == _lib.EINVAL
    assert call(ws.data_ptr(), 100) == _lib.EINVAL
    assert call(ws.data_ptr() + 8, 1 << 19) == _lib.EINVAL
    assert call(ws.data_ptr(), 1 << 20) == 0
    # the context's own stream and scratch
    torch.cuda.synchronize()
    assert ctx.lib.pion_v_b200_fp4_scores(ctx.h, rows._ref(ctx), 100, x.data_ptr(), 0, 64, 10,
                                          out.data_ptr(), 0, 100, None, 0, 1, None) == 0
    finish(ctx)
    assert torch.isneginf(out).all()
    for bad in (lambda: ctx.lib.pion_v_b200_fp4_write(ctx.h, rows._ref(ctx), x.data_ptr(), 3, 64, 1,
                                                      None, 0, 1, 1),
                lambda: ctx.lib.pion_v_b200_fp4_write(ctx.h, rows._ref(ctx), x.data_ptr(), 0, 63, 2,
                                                      None, 0, 1, 1),
                lambda: ctx.lib.pion_v_b200_fp4_write(ctx.h, rows._ref(ctx), None, 0, 64, 1, None, 0,
                                                      1, 1),
                lambda: ctx.lib.pion_v_b200_fp4_write(ctx.h, rows._ref(ctx), x.data_ptr() + 2, 0, 64,
                                                      1, None, 0, 1, 1),
                lambda: ctx.lib.pion_v_b200_fp4_write(ctx.h, rows._ref(ctx), x.data_ptr(), 0, 64, -1,
                                                      None, 0, 1, 1),
                lambda: ctx.lib.pion_v_b200_fp4_write(ctx.h, rows._ref(ctx), x.data_ptr(), 0, 64, 1,
                                                      None, 0, 2, 1),
                lambda: ctx.lib.pion_v_b200_fp4_write(ctx.h, None, x.data_ptr(), 0, 64, 1, None, 0, 1,
                                                      1)):
        assert bad() == _lib.EINVAL


def test_rows_past_32_bit_offsets(ctx):
    """A store of 4.6 GB of codes, almost all of it empty: rows near its end are written, read
    and found."""
    import pion_b200
    n = 6_000_000
    rows = pion_b200.FP4Rows(n, 1536, "nv")
    x, q = mixture_np(300, 1536, 4, seed=3, n_queries=5)
    slots = np.concatenate([np.arange(200) * 7, n - 1 - 5 * np.arange(100)])
    assert slots[-1] * 768 > 2 ** 32
    rows.write(ctx, torch.from_numpy(x).cuda(), slots=slots)
    codes, bits, g = plain.quantise(x, "nv")
    want = (plain.values(codes, bits, "nv")[:, :1536] * g[:, None].astype(np.float64))
    got = rows.read(ctx, slots=slots).cpu().numpy()
    assert np.array_equal(got, want.astype(np.float32))
    order = np.argsort(slots)
    s, _ = plain.products(q.astype(np.float64), x[order].astype(np.float64), "nv")
    wi, wv = plain.best(s, 20)
    for nq in (1, 5):
        ids, sc = pion_b200.FlatFP4Index(ctx, rows).search(torch.from_numpy(q[:nq]).cuda(), 20)
        assert np.array_equal(ids.cpu().numpy(), slots[order][wi[:nq]])
        assert np.array_equal(sc.cpu().numpy(), wv[:nq])
    finish(ctx)


def test_empty_stores_and_calls(ctx):
    import pion_b200
    rows = pion_b200.quantize_rows_fp4(ctx, torch.zeros((0, 40), device="cuda"))
    q = torch.ones((2, 40), device="cuda")
    ids, sc = pion_b200.FlatFP4Index(ctx, rows).search(q, 3)
    assert (ids == -1).all() and torch.isneginf(sc).all()
    assert pion_b200.fp4_scores(ctx, rows, q).shape == (2, 0)
    assert rows.read(ctx).shape == (0, 40)
    rows = pion_b200.FP4Rows(5, 40)
    rows.write(ctx, q[:0])
    assert pion_b200.fp4_scores(ctx, rows, q[:0]).shape == (0, 5)
    ids, sc = pion_b200.FlatFP4Index(ctx, rows).search(q[:0], 3)
    assert ids.shape == (0, 3)
    ids, sc = pion_b200.FlatFP4Index(ctx, rows).search(np.ones((2, 40), np.float32), 3)
    assert (ids == -1).all()
    finish(ctx)


def test_host_arrays(ctx):
    import pion_b200
    x, q = mixture_np(9000, 200, 30, seed=1, n_queries=20)
    rows = pion_b200.quantize_rows_fp4(ctx, x, "mx")
    check_store(rows, np.arange(9000), x, "mx")
    check_knn(ctx, rows, q, q.astype(np.float64), x.astype(np.float64), "mx", 10)
    s = pion_b200.fp4_scores(ctx, rows, q)
    d = pion_b200.fp4_scores(ctx, rows, torch.from_numpy(q).cuda())
    assert isinstance(s, np.ndarray) and np.array_equal(s, d.cpu().numpy())
    rows.write(ctx, q, slots=np.arange(20) * 3)
    check_store(rows, np.arange(20) * 3, q, "mx")
    rows.write(ctx, x[::-1][:50, ::1], start=100)          # a view with negative strides
    check_store(rows, np.arange(100, 150), x[::-1][:50], "mx")


def test_large_batches_are_searched_in_chunks(ctx):
    import pion_b200
    x, q = mixture_np(9000, 64, 30, seed=2, n_queries=4500)
    rows = pion_b200.quantize_rows_fp4(ctx, x, "nv")
    check_knn(ctx, rows, torch.from_numpy(q).cuda(), q.astype(np.float64), x.astype(np.float64),
              "nv", 3)


def test_captured_and_replayed(ctx):
    """Write, read, scores and search in a graph; replays see new inputs; a second graph of the
    same context and eager calls between replays do not disturb it."""
    import pion_b200
    x, q = mixture_np(9000, 256, 30, seed=3, n_queries=48)
    rows = pion_b200.quantize_rows_fp4(ctx, x, "nv")
    ix = pion_b200.FlatFP4Index(ctx, rows)
    tq = torch.from_numpy(q).cuda()
    new = torch.zeros((4, 256), device="cuda")
    slots = torch.zeros(4, dtype=torch.int64, device="cuda")
    sq = tq[:16].clone()

    def step():
        rows.write(ctx, new, slots=slots)
        return (*ix.search(sq, 10), pion_b200.fp4_scores(ctx, rows, sq), rows.read(ctx, slots=slots))

    slots.copy_(torch.arange(4))
    new.copy_(torch.from_numpy(x[:4]))
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    x = x.copy()
    for i in range(4):
        at = [7 * i, 100 + i, 7 * i, 8999 - i]            # a repeated slot: the last row wins
        vals = q[20 + 4 * i:24 + 4 * i]
        slots.copy_(torch.tensor(at))
        new.copy_(torch.from_numpy(vals))
        sq.copy_(tq[i:i + 16])
        x[at] = vals
        x[at[2]] = vals[2]
        g, out = graphs[i % 2]
        g.replay()
        ix.search(tq[:33], 64)
        torch.cuda.synchronize()
        want, _ = plain.products(q[i:i + 16].astype(np.float64), x.astype(np.float64), "nv")
        wi, wv = plain.best(want, 10)
        assert np.array_equal(out[0].cpu().numpy(), wi)
        assert np.array_equal(out[1].cpu().numpy(), wv)
        eager = pion_b200.fp4_scores(ctx, rows, sq)
        assert torch.equal(out[2], eager)
        assert torch.equal(out[3], rows.read(ctx, slots=slots))


def test_other_streams_and_contexts(ctx):
    import pion_b200
    x, q = mixture_np(20000, 128, 30, seed=9, n_queries=70)
    rows = pion_b200.quantize_rows_fp4(ctx, x, "mx")
    want, _ = plain.products(q.astype(np.float64), x.astype(np.float64), "mx")
    wi, wv = plain.best(want, 10)
    tq = torch.from_numpy(q).cuda()
    torch.cuda.synchronize()
    other = pion_b200.Context(0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(5):
        for c, s in ((ctx, streams[0]), (other, streams[1])):
            with torch.cuda.stream(s):
                outs.append(pion_b200.FlatFP4Index(c, rows).search(tq, 10))
    torch.cuda.synchronize()
    for ids, sc in outs:
        assert np.array_equal(ids.cpu().numpy(), wi) and np.array_equal(sc.cpu().numpy(), wv)
    other.close()


def test_ingest_search_and_rerank_together(ctx):
    """As they are used: rows arrive and are written in 4 bits beside the FP32 rows, a query
    takes a shortlist of 64 from the 4-bit rows, and the FP32 rows rank it exactly."""
    import pion_b200
    x, q = mixture_np(30000, 1536, 64, seed=21, n_queries=50)
    tx, tq = torch.from_numpy(x).cuda(), torch.from_numpy(q).cuda()
    f32 = pion_b200.FlatF32Index(ctx, tx)
    cos = 1.0 - (x.astype(np.float64) @ q.T.astype(np.float64)).T
    for fmt in ("nv", "mx"):
        rows = pion_b200.FP4Rows(30000, 1536, fmt)
        for a in range(0, 30000, 10000):
            rows.write(ctx, tx[a:a + 10000], start=a)
        ids, sc = pion_b200.FlatFP4Index(ctx, rows).search(tq, 64)
        want, _ = plain.products(q.astype(np.float64), x.astype(np.float64), fmt)
        short, _ = plain.best(want, 64)
        assert np.array_equal(ids.cpu().numpy(), short)
        got, scores = f32.merge_delta(tq, 30000, ids, sc, 10)
        finish(ctx)
        # the ten nearest of the shortlist: float32 distances of unit vectors, 1536 terms
        got, scores = got.cpu().numpy(), scores.cpu().numpy()
        mine = np.take_along_axis(cos, short, 1)
        tol = 1536 * 2.0 ** -24 * 2
        assert np.abs(np.take_along_axis(cos, got, 1) - scores).max() <= tol
        assert np.abs(np.sort(mine, axis=1)[:, :10] - scores).max() <= tol
