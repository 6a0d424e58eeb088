"""Ends of groups in the weight gradient: the last stage of a group's rows also holds rows of the next one, which both CTAs of a pair
clear before the pair's products read them."""
import pytest
import torch

from tests import grouped_helpers as H

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k,n", [(512, 512), (256, 264), (40, 24)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_of_the_next_group_are_cleared_in_both_operands(ctx, k, n, bad):
    """400 groups that end inside a stage, every second one spoiled: many turns of each stage, on every pair."""
    counts = [1 + (37 * g) % 131 for g in range(400)]
    offsets, rows = H.offsets_of(counts), sum(counts)
    A, dC = H.normal((rows, k), torch.bfloat16, 1), H.normal((rows, n), torch.bfloat16, 2)
    B = torch.empty((400, k, n), dtype=torch.bfloat16, device="cuda")
    for g, lo, hi in H.spans(offsets)[1::2]:
        A[lo:hi], dC[lo:hi] = bad, bad
    exact, size = H.weight_gradient(offsets, A, dC, False, B)
    for _ in range(20):
        _, dB = ctx.grouped_mm_grad(offsets, A, B, dC, need_dA=False)
        H.assert_rounded_sum(dB[::2], exact[::2], size[::2], max(counts))
        assert not bool(dB[1::2].isfinite().any())
    assert ctx.device_status() == 0
