"""4-bit calls in forms beside the common ones."""
import numpy as np
import pytest
import torch

import fp4_plain as plain

pytestmark = pytest.mark.gpu


def test_launches_are_counted_as_they_are_made(ctx):
    """Few rows are written without the pass that claims their slots."""
    import pion_b200
    rows = pion_b200.FP4Rows(3000, 64, "nv")
    for n, with_slots, want in ((1, True, 1), (1024, True, 1), (1025, True, 2), (1025, False, 1)):
        x = torch.zeros((n, 64), device="cuda")
        slots = torch.arange(n, device="cuda") if with_slots else None
        before = ctx.launches
        rows.write(ctx, x, slots=slots)
        assert ctx.launches - before == want
    torch.cuda.synchronize()
    ctx.sync()


def best_time(f, runs=5, calls=10):
    """The least of some mean times of a call, in us."""
    times = []
    for _ in range(runs + 1):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        torch.cuda.synchronize()
        a.record()
        for _ in range(calls):
            f()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) / calls * 1e3)
    return min(times[1:])


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("n", [2500, 16000])
def test_few_rows_among_many_empty_slots(ctx, fmt, n):
    """A store searched at its capacity while it holds fewer than k rows: they are found, and the
    empty slots are not scored one by one (16000 of them took 37 times as long as as many rows)."""
    import pion_b200
    rng = np.random.default_rng(n)
    x = torch.from_numpy(rng.standard_normal((n, 4096)).astype(np.float32)).cuda()
    full = pion_b200.quantize_rows_fp4(ctx, x, fmt)
    few = pion_b200.FP4Rows(n, 4096, fmt)
    at = [7, n // 2, n - 1]
    few.write(ctx, x[at], slots=at)
    ix = pion_b200.FlatFP4Index(ctx, few)
    q = x[at][:2] + 0.1
    ids, sc = ix.search(q, 10)
    all_ids, all_sc = pion_b200.FlatFP4Index(ctx, full).search(q, 10)
    torch.cuda.synchronize()
    ctx.sync()
    assert ids[:, 0].tolist() == at[:2] == all_ids[:, 0].tolist()
    assert torch.equal(sc[:, 0], all_sc[:, 0])
    for row in ids.tolist():
        assert sorted(row[:3]) == sorted(at) and row[3:] == [-1] * 7
    assert torch.isneginf(sc[:, 3:]).all()
    a = best_time(lambda: ix.search(q, 10))
    b = best_time(lambda: pion_b200.FlatFP4Index(ctx, full).search(q, 10))
    print(f"{fmt} {n} slots: 3 rows {a:.0f} us, full {b:.0f} us")
    assert a < 4 * b


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_host_arrays_of_every_kind(ctx, fmt):
    """float16, float64 and bfloat16 rows in host memory, inside wider buffers, read-only, and lists:
    what the same rows on the GPU give."""
    import pion_b200
    rng = np.random.default_rng(31)
    wide = rng.standard_normal((600, 90))
    wide.flags.writeable = False

    def answers(x, q):
        rows = pion_b200.quantize_rows_fp4(ctx, x, fmt)
        ids, sc = pion_b200.FlatFP4Index(ctx, rows).search(q, 7)
        s = pion_b200.fp4_scores(ctx, rows, q)
        torch.cuda.synchronize()
        ctx.sync()
        back = rows.read(ctx)
        return [torch.as_tensor(np.asarray(a.cpu() if torch.is_tensor(a) else a))
                for a in (ids, sc, s, back)]

    for host, dev in ((wide.astype(np.float16), torch.float16), (wide, torch.float32),
                      (torch.from_numpy(wide.copy()).bfloat16(), torch.bfloat16),
                      (wide.astype(np.float32)[::2], torch.float32)):
        x, q = host[:, 5:82], host[::31, 5:82]
        tx = torch.as_tensor(np.ascontiguousarray(x)) if not torch.is_tensor(x) else x
        want = answers(tx.to(dev).cuda(), tx[::31].to(dev).cuda())
        for a, b in zip(answers(x, q), want):
            assert torch.equal(a.float(), b.float())
    rows = pion_b200.FP4Rows(3, 4, fmt)
    rows.write(ctx, [[1.0, 2.0, -3.0, 0.5]], slots=[2])
    codes, bits, g = plain.quantise([[1.0, 2.0, -3.0, 0.5]], fmt)
    want = (plain.values(codes, bits, fmt)[:, :4] * g[:, None].astype(np.float64)).astype(np.float32)
    assert np.array_equal(rows.read(ctx, slots=(2,)).cpu().numpy(), want)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("stall", ["1", "2", "3"])
def test_waits_that_run_out_in_either_cta(ctx, monkeypatch, fmt, stall):
    """The issuing warp, or the copies of one CTA of a pair, wait for what never comes: the CTAs have
    copied different numbers of stages when they give up; they settle what is in flight, the call
    reports it, and the next is right."""
    import time

    import pion_b200
    rng = np.random.default_rng(17)
    x = torch.from_numpy(rng.standard_normal((30000, 1000)).astype(np.float32)).cuda()
    rows = pion_b200.quantize_rows_fp4(ctx, x, fmt)
    ix = pion_b200.FlatFP4Index(ctx, rows)
    q = x[:600] + 0.1
    for nq in (1, 600):
        want = pion_b200.fp4_scores(ctx, rows, q[:nq])
        ids, sc = ix.search(q[:nq], 10)
        torch.cuda.synchronize()
        ctx.sync()
        ctx.set_wait_budget(1_000_000)
        monkeypatch.setenv("PION_B200_TEST_STALL", stall)
        try:
            for call in (lambda: pion_b200.fp4_scores(ctx, rows, q[:nq]), lambda: ix.search(q[:nq], 10)):
                t0 = time.perf_counter()
                call()
                torch.cuda.synchronize()
                assert time.perf_counter() - t0 < 1.5      # no wait of the drain's own 2 s ran out
                with pytest.raises(pion_b200.PionError) as e:
                    ctx.sync()
                assert e.value.code == -11
        finally:
            monkeypatch.delenv("PION_B200_TEST_STALL")
            ctx.set_wait_budget(0)
        assert torch.equal(pion_b200.fp4_scores(ctx, rows, q[:nq]), want)
        again = ix.search(q[:nq], 10)
        assert torch.equal(again[0], ids) and torch.equal(again[1], sc)
        torch.cuda.synchronize()
        ctx.sync()


def test_host_memory_is_refused_while_capturing(ctx):
    """The refusal leaves the capture, the context and torch as they were."""
    import pion_b200
    rng = np.random.default_rng(2)
    x = rng.standard_normal((300, 64)).astype(np.float32)
    rows = pion_b200.quantize_rows_fp4(ctx, x, "nv")
    ix = pion_b200.FlatFP4Index(ctx, rows)
    tq = torch.from_numpy(x[:4]).cuda()
    want = [t.clone() for t in ix.search(tq, 5)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for bad in (lambda: rows.write(ctx, x[:3], start=0), lambda: ix.search(x[:4], 5),
                    lambda: pion_b200.fp4_scores(ctx, rows, x[:4])):
            with pytest.raises(pion_b200.PionError) as e:
                bad()
            assert e.value.code == -1
        out = ix.search(tq, 5)
    g.replay()
    torch.cuda.synchronize()
    ctx.sync()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    ids, sc = ix.search(x[:4], 5)
    assert np.array_equal(ids, want[0].cpu().numpy())
