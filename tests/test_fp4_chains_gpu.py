"""Calls that follow each other on one buffer without a wait between them: each kernel may start while
the ones before it run, and sees what they wrote."""
import numpy as np
import pytest
import torch

import fp4_plain as plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("dim,stride,n", [(777, 777, 64), (777, 784, 40), (1003, 1003, 1500),
                                          (33, 40, 2000), (130, 130, 7)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_read_into_a_buffer_and_written_again(ctx, fmt, dim, stride, n, dtype):
    """read(out=buf); write(buf) from one store to the next, many times: tails and unaligned rows of
    the one buffer are new every time."""
    import pion_b200
    rng = np.random.default_rng(dim + n)
    sources = [pion_b200.quantize_rows_fp4(
        ctx, torch.from_numpy(rng.standard_normal((n, dim)).astype(np.float32)).cuda(), fmt)
        for _ in range(3)]
    slots = [torch.randperm(n + 3, device="cuda")[:n] for _ in range(3)]
    buf = torch.empty((n, stride), dtype=dtype, device="cuda")[:, :dim]
    want = [s.read(ctx, dtype=dtype) for s in sources]
    targets = [pion_b200.FP4Rows(n + 3, dim, fmt) for _ in range(24)]
    torch.cuda.synchronize()
    for i, t in enumerate(targets):
        sources[i % 3].read(ctx, out=buf)
        t.write(ctx, buf, slots=slots[i % 3])
    torch.cuda.synchronize()
    ctx.sync()
    for i, t in enumerate(targets):
        at = slots[i % 3].cpu().numpy()
        codes, bits, g = plain.quantise(want[i % 3].double().cpu().numpy(), fmt)
        c = t.codes.cpu().numpy()[at]
        got = np.stack((c & 15, c >> 4), 2).reshape(n, -1)
        assert np.array_equal(np.where(got == 8, 0, got), np.where(codes == 8, 0, codes))
        assert np.array_equal(t.row_scale.cpu().numpy()[at], g)
        assert not t.claim.any()
