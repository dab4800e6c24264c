"""Sums of 4-bit products that float64 cannot hold, or float32 cannot, against integers.

The definition here is in Python's integers: a score is the exact ((sum) g_r) g_t rounded once to
float32.  ids and scores of a search are compared bit for bit."""
from fractions import Fraction

import numpy as np
import pytest
import torch

import fp4_plain as plain

pytestmark = pytest.mark.gpu


def to_f32(x: Fraction) -> np.float32:
    """x rounded to nearest, ties to even, through integers."""
    if x == 0:
        return np.float32(0)
    n, d = abs(x.numerator), x.denominator
    e = n.bit_length() - d.bit_length()          # 2^(e-1) < n / d < 2^(e+1)
    if (n << max(-e, 0)) < (d << max(e, 0)):
        e -= 1
    e = max(e, -126) - 23                        # the last bit's weight
    n, d = n << max(-e, 0), d << max(e, 0)
    q, r = divmod(n, d)
    q += 2 * r > d or (2 * r == d and q & 1)
    v = np.inf if q.bit_length() + e > 128 else np.float32(np.ldexp(float(q), e))
    return np.float32(-v if x < 0 else v)


def integers(codes, bits, fmt):
    """Rows as Python integers [n, dp] in units of 2^-128 (mx) or 2^-10 (nv), exactly."""
    twice = np.array([0, 1, 2, 3, 4, 6, 8, 12] + [0, -1, -2, -3, -4, -6, -8, -12], dtype=object)
    if fmt == "mx":
        s = np.array([1 << b for b in range(256)], dtype=object)
    else:
        s = np.array([int(v * 512) for v in plain.E4M3] + [0] * 129, dtype=object)
    return twice[codes] * np.repeat(s[bits], plain.BLOCK[fmt], axis=1)


def exact_scores(q, x, fmt):
    """float32 [nq, n] of raw queries and rows, every row finite."""
    qc, qb, qg = plain.quantise(q, fmt)
    rc, rb, rg = plain.quantise(x, fmt)
    a, b = integers(qc, qb, fmt), integers(rc, rb, fmt)
    unit = Fraction(1, 2 ** (256 if fmt == "mx" else 20))
    out = np.zeros((len(q), len(x)), np.float32)
    for t in range(len(q)):
        at = np.flatnonzero(a[t])
        s = (b[:, at] * a[t, at]).sum(1) if len(at) else np.zeros(len(x), dtype=object)
        for r in range(len(x)):
            out[t, r] = to_f32(Fraction(int(s[r])) * unit * Fraction(float(rg[r])) *
                               Fraction(float(qg[t])))
    return out


def test_rounding_of_the_definition():
    for v in (1.0, -3.5, 2.0 ** -149, 2.0 ** -126, float(np.finfo(np.float32).max)):
        assert to_f32(Fraction(v)) == np.float32(v)
    half = Fraction(1, 2 ** 24)
    assert to_f32(1 + half) == 1 and to_f32(1 + half + Fraction(1, 2 ** 90)) > 1
    assert to_f32(1 + 3 * half) == np.float32(1 + 2.0 ** -22)
    assert to_f32(Fraction(2) ** 128) == np.inf and to_f32(Fraction(1, 2 ** 150)) == 0
    assert to_f32(Fraction(3, 2 ** 151)) == np.float32(2.0 ** -149)


def check(ctx, q, x, fmt, k, copies=1):
    """A search of `copies` times the rows x, with the lowest ids of equal scores."""
    import pion_b200
    q, x = np.asarray(q, np.float32), np.asarray(x, np.float32)
    s = np.tile(exact_scores(q.astype(np.float64), x.astype(np.float64), fmt), (1, copies))
    wi, wv = plain.best(s, k)
    rows = pion_b200.quantize_rows_fp4(ctx, torch.from_numpy(x).cuda().repeat(copies, 1), fmt)
    for nq in {1, len(q)}:
        ids, sc = pion_b200.FlatFP4Index(ctx, rows).search(torch.from_numpy(q[:nq]).cuda(), k)
        torch.cuda.synchronize()
        ctx.sync()
        assert np.array_equal(ids.cpu().numpy(), wi[:nq])
        assert np.array_equal(sc.cpu().numpy().view(np.uint32), wv[:nq].view(np.uint32))


# rows of few, of more than are scored at once, and of so many that thresholds are sampled
SIZES = [(200, 1), (250, 12), (250, 80)]


@pytest.mark.parametrize("n,copies", SIZES)
@pytest.mark.parametrize("blocks", [4, 5, 48, 256])
def test_blocks_that_cancel_mx(ctx, n, copies, blocks):
    """Rows made of the same blocks in another order, among them pairs that cancel and are 2^60
    (or 2^150 and 2^90) times the rest: all sums are equal, and the lowest ids are the best."""
    rng = np.random.default_rng(blocks + n)
    for powers in ([60, 0], [60, 57, 0], [100, 40, 0, -30], [25, 0]):
        x = np.zeros((n, 32 * blocks))
        for i in range(n):
            v = [s * 2.0 ** p for p in powers[:-1] for s in (1, -1)][:blocks - 1] + [2.0 ** powers[-1]]
            at = rng.permutation(blocks)[:len(v)] * 32 + rng.integers(0, 32, len(v))
            x[i, at] = v
        check(ctx, np.ones((3, 32 * blocks)), x, "mx", 10, copies)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("n,copies", SIZES)
def test_random_blocks_of_far_magnitudes(ctx, fmt, n, copies):
    """Random codes in blocks of magnitudes from the least to the largest: sums whose bits span up
    to 500, cancel or not, and are rounded once."""
    rng = np.random.default_rng(n + copies)
    for dim, span in ((100, 12), (640, 30), (1000, 58), (512, 31), (512, 33)):
        top = span if fmt == "mx" else min(span, 17)
        x = rng.integers(-6, 7, (n, dim)) * np.exp2(rng.integers(-top, top + 1, (n, dim // 4))).repeat(4, 1)
        q = rng.integers(-6, 7, (5, dim)) * np.exp2(rng.integers(-top, top + 1, (5, dim // 4))).repeat(4, 1)
        x[1::2, dim // 2:] = -x[1::2, dim // 2 - 1::-1][:, :dim - dim // 2]   # near-cancelling halves
        q[1::2, dim // 2:] = q[1::2, dim // 2 - 1::-1][:, :dim - dim // 2]
        check(ctx, q, x, fmt, 10, copies)


@pytest.mark.parametrize("n,copies", SIZES)
def test_blocks_that_cancel_nv(ctx, n, copies):
    """Products whose sum needs 56 bits: blocks of +-448 * 6 that cancel around one product of
    2^-20."""
    rng = np.random.default_rng(n)
    dim = 8192
    q = np.full((3, dim), 2688.0)
    q[:, 4000:4016] = 0
    q[:, 4000], q[:, 4003] = 6 * 2.0 ** -9, 2.0 ** -10    # a block of the least scale, 2^-9
    x = np.zeros((n, dim))
    for i in range(n):
        order = rng.permutation(510)
        at = np.delete(np.arange(512), [250, 511])[order]
        sign = np.zeros(512)
        if i % 2:   # by halves of the parity of the 32-element block, else at random
            at = np.array(sorted(np.delete(np.arange(512), [250, 511]), key=lambda b: (b // 2) % 2))
        sign[at[:255]], sign[at[255:]] = 1, -1
        x[i] = np.repeat(sign, 16) * 2688.0
        x[i, 4000:4016] = 0
        x[i, 4001], x[i, 4003] = 6 * 2.0 ** -9, 2.0 ** -10 * rng.choice([1, 2])
    check(ctx, q, x, "nv", 10, copies)


@pytest.mark.parametrize("n,copies", SIZES)
def test_products_past_float32_that_cancel(ctx, n, copies):
    """Products of +-2^200 and 2^120 that cancel around ones between 2^-100 and 2^60."""
    rng = np.random.default_rng(n + 3)
    q = np.repeat(2.0 ** np.array([100] * 16 + [60] * 16 + [-60] * 16 + [30] * 16), 32)[None].repeat(3, 0)
    x = np.zeros((n, 2048))
    for i in range(n):
        big, mid = rng.permutation(16) * 32, 512 + rng.permutation(16) * 32
        x[i, big[:12]] = 2.0 ** 100 * np.array([1, -1, 3, -3, 2, -2, 6, -6, 1, -1, 1, -1])
        x[i, mid[:6]] = 2.0 ** 60 * np.array([1, -1, 4, -4, 0.5, -0.5])
        x[i, 1024 + rng.integers(0, 512)] = 2.0 ** -40 * (1 + i % 2)
        x[i, 1536 + rng.integers(0, 512)] = 2.0 ** 30 if i % 5 == 0 else 0
    check(ctx, q, x, "mx", 10, copies)


def test_sums_that_leave_float32_are_no_empty_slots(ctx):
    """-inf is an empty row's or query's score; a live one's sum past float32 is infinite by the sign
    with which it left float32."""
    import pion_b200
    x = np.zeros((6, 256), np.float32)
    q = np.zeros((4, 256), np.float32)
    q[0, ::32] = 2.0 ** 100
    q[1, ::32] = 1
    q[3, 0] = np.nan
    x[0, ::32] = 2.0 ** 100 * np.array([1, 1, -1, -1] * 2)
    x[1, ::32] = 2.0 ** 100
    x[2, ::32] = -2.0 ** 100
    x[3, 0] = np.inf
    x[4, ::32] = 1
    rows = pion_b200.quantize_rows_fp4(ctx, torch.from_numpy(x).cuda(), "mx")
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        s = pion_b200.fp4_scores(ctx, rows, torch.from_numpy(q).cuda(), dtype=dtype)
        torch.cuda.synchronize()
        ctx.sync()
        s = s.double().cpu().numpy()
        assert s[0, 0] == np.inf and s[0, 1] == np.inf and s[0, 2] == -np.inf
        assert np.isneginf(s[:, 3]).all() and np.isneginf(s[3]).all()
        assert s[1, 0] == 0 and (s[2, [0, 1, 2, 4, 5]] == 0).all() and s[1, 4] == 8
        assert (s[:3, 5] == 0).all()
