"""4-bit calls in forms beside the common ones."""
import numpy as np
import pytest
import torch

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
