"""A call that the GPU's memory or a launch refuses leaves nothing behind for the calls after it."""
import pytest
import torch

from sparsewave_b200 import SparseWaveError, _lib
from tests import grouped_helpers as H

pytestmark = pytest.mark.gpu


def test_a_call_refused_for_lack_of_memory_fails_alone(ctx):
    """Weights of one column have to be copied to rows of 16 bytes, eight times their 34 GB: more than the GPU has."""
    inner = 2 ** 31 - 1024
    A = torch.empty((1, inner), dtype=torch.bfloat16, device="cuda")
    B = torch.empty((8, inner, 1), dtype=torch.bfloat16, device="cuda")
    assert B.numel() * 16 > torch.cuda.get_device_properties(0).total_memory
    X, W = H.normal((20, 31), torch.bfloat16, 1), H.normal((2, 31, 40), torch.bfloat16, 2)
    offsets = H.offsets_of([5, 15])
    for _ in range(2):
        with pytest.raises(SparseWaveError) as e:
            ctx.grouped_mm(H.offsets_of([1, 0, 0, 0, 0, 0, 0, 0]), A, B)
        assert e.value.status == _lib.SWB_ERR_CUDA and "memory" in str(e.value)
        C = ctx.grouped_mm(offsets, X, W)
        exact, size = H.grouped_mm(offsets, X, W, False)
        H.assert_rounded_sum(C, exact, size, 31)
    with pytest.raises(SparseWaveError):
        ctx.grouped_mm(H.offsets_of([1, 0, 0, 0, 0, 0, 0, 0]), A, B)
    assert float(torch.ones(3, device="cuda").sum()) == 3.0  # torch's own checks see no error either
    torch.cuda.synchronize()
    Q, scales = ctx.fp8_quantize_rows(X)
    q, s = H.quantize_rows(X)
    assert torch.equal(Q.view(torch.uint8), q.view(torch.uint8)) and torch.equal(scales, s)


def test_a_workspace_that_cannot_be_had_fails_alone(ctx):
    """The same for the calls on host buffers, whose device workspace is asked for before anything is read."""
    lib, cols, n = _lib.load(), 2 ** 31 - 1, 64
    assert cols * n * 4 > 2 * torch.cuda.get_device_properties(0).total_memory
    row_ptr, C = torch.zeros(2, dtype=torch.int32), torch.zeros((1, n))
    options = _lib.SwbOptions()
    lib.swb_options_default(options)
    st = lib.swb_spmm_host(ctx._ctx, options, 1, cols, 0, n, row_ptr.data_ptr(), None, None, C.data_ptr(), C.data_ptr())
    assert st == _lib.SWB_ERR_CUDA and b"out of memory" in lib.swb_last_error(ctx._ctx)
    assert float(torch.ones(3, device="cuda").sum()) == 3.0
    got = ctx.spmv("", torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"),
                   torch.ones(1, device="cuda"), torch.full((1,), 5.0, device="cuda"))
    assert got.tolist() == [5.0]
