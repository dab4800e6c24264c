"""Products whose float32 sums are exact, again and again: every row of both CTAs of a pair and every
query of both halves of a tile has to be there when it is multiplied."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("n,dim,nq", [(20000, 1536, 1), (70001, 256, 1000), (9000, 5000, 300),
                                      (40000, 128, 16)])
def test_products_of_small_integers(ctx, fmt, n, dim, nq):
    """Elements of the code grid with a 6 in every block (and 2688 = 448 * 6 in every row of NV,
    whose scales are then small integers): sums below 2^24 units."""
    import pion_b200
    rng = np.random.default_rng(n + dim)

    def grid(rows):
        x = rng.choice([0, 0, 0, 1, -1, 2, -2, 3, -4], (rows, dim)).astype(np.float32)
        x[:, 5::16] = rng.choice([6, -6], x[:, 5::16].shape)
        return x

    x, q = grid(n), grid(nq)
    tx, tq = torch.from_numpy(x).cuda(), torch.from_numpy(q).cuda()
    want = (tq.double() @ tx.double().T).float()
    assert want.abs().max() * 4 < 2 ** 24
    if fmt == "nv":       # g = 6 / 2688, scales 448: elements are exact in units of 448 g
        unit = np.float32(6) / np.float32(2688)
        want = ((tq.double() @ tx.double().T) * 448.0 ** 2).float() * float(unit) * float(unit)
    rows = pion_b200.quantize_rows_fp4(ctx, tx, fmt)
    flush = torch.empty(1 << 26, dtype=torch.float32, device="cuda")
    for i in range(6):
        if i % 2:
            flush.zero_()                       # rows from HBM, then from L2
        got = pion_b200.fp4_scores(ctx, rows, tq)
        torch.cuda.synchronize()
        ctx.sync()
        assert torch.equal(got, want)
