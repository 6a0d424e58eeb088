"""One gradient without the other's operand: B takes no part in its own gradient, nor A in its."""
import pytest
import torch

from sparsewave_b200 import SparseWaveError, _lib
from tests import grouped_helpers as H

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts,k,n", [([20, 0, 150, 3], 256, 128), ([5], 33, 50), ([5000], 128, 136), ([0, 0], 16, 24)])
@pytest.mark.parametrize("transpose_b", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_same_as_with_both(ctx, counts, k, n, transpose_b, dtype):
    offsets, rows, groups = H.offsets_of(counts), sum(counts), len(counts)
    A, dC = H.normal((rows, k), dtype, 1), H.normal((rows, n), dtype, 2)
    B = H.normal((groups, n, k) if transpose_b else (groups, k, n), dtype, 3, k ** -0.5)
    dA, dB = ctx.grouped_mm_grad(offsets, A, B, dC, transpose_b=transpose_b)
    none, only_b = ctx.grouped_mm_grad(offsets, A, None, dC, transpose_b=transpose_b, need_dA=False)
    assert none is None and only_b.dtype == dtype and torch.equal(only_b, dB)
    only_a, none = ctx.grouped_mm_grad(offsets, None, B, dC, transpose_b=transpose_b, need_dB=False)
    assert none is None and only_a.dtype == dtype and torch.equal(only_a, dA)
    given = torch.full_like(B, 7.0)
    assert ctx.grouped_mm_grad(offsets, A, None, dC, None, given, transpose_b=transpose_b, need_dA=False)[1] is given
    assert torch.equal(given, dB)


def test_refusals(ctx):
    A, B = H.normal((8, 16), torch.bfloat16, 1), H.normal((2, 16, 24), torch.bfloat16, 2)
    dC, offsets = H.normal((8, 24), torch.bfloat16, 3), H.offsets_of([4, 4])
    for call in (lambda: ctx.grouped_mm_grad(offsets, None, B, dC), lambda: ctx.grouped_mm_grad(offsets, A, None, dC),
                 lambda: ctx.grouped_mm_grad(offsets, None, B, dC, need_dA=False), lambda: ctx.grouped_mm_grad(offsets, A, None, dC, need_dB=False),
                 lambda: ctx.grouped_mm_grad(offsets, None, None, dC, need_dA=False, need_dB=False),
                 lambda: ctx.grouped_mm_grad(offsets, None, B, dC.float(), need_dB=False),
                 lambda: ctx.grouped_mm_grad(offsets, None, B.half(), dC, need_dB=False)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: ctx.grouped_mm_grad(offsets[:1], A, None, dC, need_dA=False), lambda: ctx.grouped_mm_grad(offsets[:0], A, None, dC, need_dA=False),
                 lambda: ctx.grouped_mm_grad(offsets, A, None, dC[:7], need_dA=False),
                 lambda: ctx.grouped_mm_grad(offsets, None, B, dC[:, :23].contiguous(), need_dB=False),
                 lambda: ctx.grouped_mm_grad(offsets[:2], None, B, dC, need_dB=False),
                 lambda: ctx.grouped_mm_grad(offsets, A, None, dC, None, torch.empty_like(B[:1]), need_dA=False)):
        with pytest.raises(SparseWaveError) as e:
            call()
        assert e.value.status == _lib.SWB_ERR_INVALID_SHAPE
